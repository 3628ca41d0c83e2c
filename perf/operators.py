"""Decoding from a tree of drafted tokens, operator by operator: the tree's rotation and cache append,
its attention over the cache, the verification of its tokens against the target's probabilities,
and the gather that keeps the accepted rows of a cache. With `own` false each runs in a plain form
of elementary torch operations; with `own` true it runs through this library's entry points.

A tree has `nodes` tokens. Node 0 is the last token that was decided (not in the cache yet), the
others are drafts; a node's parent has a lower number. Position past + i of the caches holds node i."""
import math
import os
import sys

import numpy as np
import torch

own = False

HD = 64            # head_dim of the f16 caches
THETA = 1e6        # rope base of the Qwen2.5-0.5B shape
VOCAB = 151936     # its vocabulary
LAYERS = 24        # its decoder layers


def listed():
    return [
        # The rotation and append of one layer's drafts: a chain of five, the smallest call, and a
        # wide tree behind a long context.
        {"name": "append-5-at-1024", "kind": "append", "nodes": 5, "past": 1024, "width": 1, "heads": 14, "kv": 2},
        {"name": "append-256-at-8000", "kind": "append", "nodes": 256, "past": 8000, "width": 4, "heads": 14, "kv": 2},
        # One layer's attention of a short chain of drafts in a short chat: latency alone.
        {"name": "attn-5-at-123", "kind": "attn", "nodes": 5, "past": 123, "width": 1, "heads": 14, "kv": 2},
        # The ordinary tree at the context of the decode benchmark, and a larger one further on.
        {"name": "attn-16-at-1024", "kind": "attn", "nodes": 16, "past": 1024, "width": 3, "heads": 14, "kv": 2},
        {"name": "attn-63-at-4097", "kind": "attn", "nodes": 63, "past": 4097, "width": 4, "heads": 14, "kv": 2},
        # A full tree at the long end of the context, and the widest one there.
        {"name": "attn-64-at-32700", "kind": "attn", "nodes": 64, "past": 32700, "width": 4, "heads": 14, "kv": 2},
        {"name": "attn-256-at-32512", "kind": "attn", "nodes": 256, "past": 32512, "width": 4, "heads": 14, "kv": 2},
        # Verification: greedy decoding over a chain; a tree whose tokens were looked up, not sampled;
        # a sampled tree with the draft model's probabilities.
        {"name": "verify-greedy-5", "kind": "verify", "how": "greedy", "nodes": 5, "width": 1, "depth": 4, "vocab": VOCAB},
        {"name": "verify-lookup-64", "kind": "verify", "how": "lookup", "nodes": 64, "width": 4, "depth": 8, "vocab": VOCAB},
        {"name": "verify-sampled-tree-32", "kind": "verify", "how": "sampled", "nodes": 32, "width": 3, "depth": 6, "vocab": VOCAB},
        # The accepted rows of a tree moved together in all layers' caches, and a long cache thinned
        # out into half its positions.
        {"name": "gather-commit-6-of-64", "kind": "commit", "nodes": 64, "count": 6, "past": 1024, "layers": LAYERS, "kv": 2},
        {"name": "gather-16384-of-32768", "kind": "thin", "keep": 16384, "past": 32768, "layers": LAYERS, "kv": 2},
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attn", "attn", "attn", "verify", "verify", "verify", "commit", "thin"))
    heads, kv = rng.choice(((14, 2), (14, 2), (8, 2), (4, 4), (16, 1)))
    if kind in ("append", "attn"):
        return {"kind": kind, "nodes": _logint(rng, 1, 256), "past": rng.choice((0, _logint(rng, 1, 1024), _logint(rng, 1, 32512))),
                "width": rng.randint(1, 5), "heads": heads if kind == "append" else min(heads, 14), "kv": kv}
    if kind == "verify":
        how = rng.choice(("greedy", "lookup", "sampled"))
        nodes = _logint(rng, 1, 64 if how != "sampled" else 32)
        return {"kind": kind, "how": how, "nodes": nodes, "width": rng.randint(1, 4),
                "depth": min(nodes - 1, rng.randint(1, 8)), "vocab": rng.choice((VOCAB, _logint(rng, 1000, VOCAB)))}
    layers = rng.choice((1, LAYERS, rng.randint(2, 32)))
    if kind == "commit":
        nodes = _logint(rng, 8, 256)
        return {"kind": kind, "nodes": nodes, "count": rng.randint(1, min(nodes // 2, 12)), "past": _logint(rng, 1, 8192),
                "layers": layers, "kv": kv}
    past = _logint(rng, 64, 32768 * LAYERS * 2 // (kv * max(layers, LAYERS)))
    return {"kind": kind, "keep": rng.randint(1, past // 2), "past": past, "layers": layers, "kv": kv}


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _rng(seed):
    return np.random.RandomState((int(seed) * 2654435761 + 977) % (1 << 32))


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _tree(rng, nodes, width, depth=None):
    """Parents of a random tree: a chain of `depth` first, then each further node under a random
    node with fewer than `width` children; a node's number is above its parent's."""
    parent, kids = [-1], [0] * nodes
    for i in range(1, nodes):
        if depth is not None and i <= depth:
            p = i - 1
        else:
            room = [j for j in range(i) if kids[j] < width]
            p = room[0] if depth is None and rng.random_sample() < 0.5 else room[rng.randint(len(room))]
        parent.append(p)
        kids[p] += 1
    return np.array(parent, np.int32)


def _ancestors(parent):
    """bool [nodes, nodes]: node i sees itself and its ancestors; and the depths."""
    n = len(parent)
    see = np.zeros((n, n), bool)
    depth = np.zeros(n, np.int32)
    for i in range(n):
        if parent[i] >= 0:
            see[i] = see[parent[i]]
            depth[i] = depth[parent[i]] + 1
        see[i, i] = True
    return see, depth


def _pack(see):
    """uint64 words [nodes, ceil(nodes / 64)], bit j % 64 of word j / 64 = column j."""
    n = see.shape[0]
    wide = np.zeros((n, (n + 63) // 64 * 64), bool)
    wide[:, :n] = see
    return np.packbits(wide, axis=1, bitorder="little").view(np.uint64)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _vstride(capacity):
    return (capacity + 63) // 64 * 64


def _rope_tables(positions):
    inv = THETA ** (-torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv[None]
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g, rng, k = _gen(seed), _rng(seed), case["kind"]
    s = {"case": dict(case)}
    if k in ("append", "attn"):
        n, past, kv = case["nodes"], case["past"], case["kv"]
        see, depth = _ancestors(_tree(rng, n, case["width"]))
        cap = past + n
        s["q"] = _randn(g, n, case["heads"] * HD)
        if k == "append":
            s["k"], s["v"] = _randn(g, n, kv * HD), _randn(g, n, kv * HD)
            s["depth"] = _cuda(depth)
            s["cos"], s["sin"] = _rope_tables(cap)
            s["qr"] = torch.zeros_like(s["q"])
        else:
            s["mask"] = _cuda(_pack(see).view(np.int64))
            s["out"] = torch.zeros_like(s["q"])
        s["keys"] = _randn(g, kv, cap, HD, dtype=torch.float16)
        s["values"] = _randn(g, kv, HD, _vstride(cap), dtype=torch.float16)
        return s
    if k == "verify":
        # Logits with a few likely tokens, as a language model's; the drafts come from a noisy copy
        # of the target's distribution, so that some are accepted and some are not.
        n, vocab, how = case["nodes"], case["vocab"], case["how"]
        parent = _tree(rng, n, case["width"], case["depth"])
        s["parent"] = _cuda(parent)
        s["logits"] = _randn(g, n, vocab, std=2.5)
        top = torch.randint(vocab, (n, 6), generator=g, device="cuda")
        s["logits"].scatter_add_(1, top, _randn(g, n, 6, std=2.0) + 12)
        noisy = torch.softmax((s["logits"] + _randn(g, n, vocab, std=0.7)) / 0.8, 1)
        at = torch.from_numpy(np.maximum(parent, 0)).long().cuda()
        drawn = torch.multinomial(noisy[at], 1, generator=g)[:, 0]
        if how == "greedy":
            best = s["logits"][at].argmax(1)
            drawn = torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, best, drawn)
        s["tokens"] = drawn.to(torch.int32)
        s["draft"] = noisy if how == "sampled" else None
        s["temperature"] = 0.0 if how == "greedy" else 0.8
        s["uniform"] = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        s["path"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["count"], s["next"] = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
        see, _ = _ancestors(parent)
        earlier = (parent[:, None] == parent[None]) & (np.arange(n)[:, None] > np.arange(n)[None])
        s["plain"] = {"see": _cuda(see), "earlier": _cuda(earlier), "most": int(earlier.sum(1).max()) + 1,
                      "kids": _cuda((parent[None] == np.arange(n)[:, None]).sum(1, keepdims=True))}
        return s
    kv, layers, past = case["kv"], case["layers"], case["past"]
    src = past + case["nodes"] if k == "commit" else past
    if k == "commit":
        # The accepted nodes of a tree numbered level by level: each comes after the rows it moves to.
        n, count = case["nodes"], case["count"]
        rows = np.full(n, -1, np.int32)
        rows[:count] = np.concatenate(([0], count + np.sort(rng.choice(n - count, count - 1, replace=False))))
        s["count"] = _cuda(np.array([count], np.int32))
    else:
        # The first positions, the most recent ones and some of those between.
        keep = case["keep"]
        must = np.union1d(np.arange(min(4, keep)), np.arange(past - max(0, (keep - 4) // 2), past))
        rest = np.setdiff1d(np.arange(past), must)
        rows = np.sort(np.concatenate((must, rng.choice(rest, keep - len(must), replace=False)))).astype(np.int32)
    s["rows"] = _cuda(rows)
    s["keys"] = torch.empty((layers, kv, src, HD), dtype=torch.float16, device="cuda")
    s["values"] = torch.empty((layers, kv, HD, _vstride(src)), dtype=torch.float16, device="cuda")
    for i in range(layers):
        s["keys"][i], s["values"][i] = _randn(g, *s["keys"][i].shape, dtype=torch.float16), _randn(g, *s["values"][i].shape, dtype=torch.float16)
    if k == "thin":
        s["to_keys"] = torch.zeros((layers, kv, keep, HD), dtype=torch.float16, device="cuda")
        s["to_values"] = torch.zeros((layers, kv, HD, _vstride(keep)), dtype=torch.float16, device="cuda")
    return s


# ------------------------------------------------------------- plain forms --

def _unpack(mask, n):
    j = torch.arange(n, device="cuda")
    return (mask[:, j // 64] >> (j % 64)) & 1 != 0


def _plain_append(s):
    c = s["case"]
    n, past = c["nodes"], c["past"]
    at = past + s["depth"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    rot = lambda t: torch.cat((t[..., :32] * cos - t[..., 32:] * sin, t[..., 32:] * cos + t[..., :32] * sin), 2)  # noqa: E731
    s["qr"] = rot(s["q"].view(n, -1, HD)).reshape(n, -1)
    s["keys"][:, past:past + n] = rot(s["k"].view(n, -1, HD)).transpose(0, 1).half()
    s["values"][:, :, past:past + n] = s["v"].view(n, -1, HD).permute(1, 2, 0).half()
    return {"q": s["qr"], "keys": s["keys"], "values": s["values"]}


def _plain_attention(s):
    c = s["case"]
    n, past, kv, heads = c["nodes"], c["past"], c["kv"], c["heads"]
    group = heads // kv
    q = s["q"].view(n, kv, group, HD).permute(1, 2, 0, 3).reshape(kv, group * n, HD)
    score = (q @ s["keys"].float().transpose(1, 2).contiguous()).mul_(1 / math.sqrt(HD)).view(kv, group, n, past + n)
    score[..., past:].masked_fill_(~_unpack(s["mask"], n), -math.inf)
    p = score.sub_(score.amax(3, keepdim=True)).exp_()
    total = p.sum(3, keepdim=True)
    values = s["values"][:, :, :past + n].float().transpose(1, 2).contiguous()
    out = (p.view(kv, group * n, past + n) @ values).view(kv, group, n, HD) / total
    s["out"] = out.permute(2, 0, 1, 3).reshape(n, heads * HD)
    return {"out": s["out"]}


def _plain_verify(s):
    """Every node is tested against its parent's distribution as its earlier siblings leave it; the
    path follows each node's first accepted child. In 64 bits: the picks lie next to borders of sums
    over the whole vocabulary."""
    n, vocab = s["case"]["nodes"], s["case"]["vocab"]
    parent, tokens, t = s["parent"].long(), s["tokens"].long(), s["plain"]
    ids, rank, ar = torch.arange(vocab, device="cuda"), t["earlier"].sum(1), torch.arange(n, device="cuda")
    up = parent.clamp(min=0)
    logits, top = s["logits"], s["logits"].amax(1, keepdim=True)
    if s["temperature"] == 0:
        best = torch.where(logits == top, ids, vocab).amin(1)
        accept = tokens == best[up]
        rest = None
    else:
        rest = ((logits.double() - top) / s["temperature"]).exp_()
        rest /= rest.sum(1, keepdim=True)
        accept = torch.zeros(n, dtype=torch.bool, device="cuda")
        p, a = rest, torch.zeros((n, 1), dtype=torch.float64, device="cuda")
        q = None if s["draft"] is None else s["draft"].double()
        rest = p if q is not None else p.clone()
        left = torch.ones((n, 1), dtype=torch.float64, device="cuda")
        for r in range(t["most"]):  # the r-th children of all nodes at once
            mine = (rank == r) & (parent >= 0)
            x = rest[up, tokens]
            if q is None:
                accept |= mine & (s["uniform"] * left[up, 0] < x)
                rest.index_put_((up, tokens), torch.where(mine, -x, 0.0 * x), accumulate=True)
                left = rest.sum(1, keepdim=True)
            else:
                accept |= mine & (s["uniform"] * q[up, tokens] * left[up, 0] < x)
                a = torch.where(t["kids"] > r, a + left, a)
                rest = (p - a * q).clamp_(min=0)
                left = rest.sum(1, keepdim=True)
    accept &= parent >= 0
    first = accept & ~(t["earlier"] & accept[None]).any(1)
    first[0] = True
    on = ~(t["see"] & ~first[None]).any(1)
    path = torch.where(on, ar, n).sort().values
    s["count"] = on.sum().to(torch.int32).view(1)
    s["path"] = torch.where(path < n, path, -1).to(torch.int32)
    end = torch.where(on, ar, 0).amax()
    if rest is None:
        s["next"] = best[end].to(torch.int32).view(1)
    else:
        w = rest[end]
        c = w.cumsum(0)
        s["next"] = torch.where((c > s["uniform"][0] * c[-1]) & (w > 0), ids, vocab).amin().to(torch.int32).view(1)
    return {"path": s["path"], "count": s["count"], "next": s["next"]}


def _plain_commit(s):
    past, n = s["case"]["past"], s["case"]["nodes"]
    j = torch.arange(n, device="cuda")
    at = past + torch.where(j < s["count"], s["rows"].long(), j)
    s["keys"][:, :, past:past + n] = s["keys"][:, :, at]
    s["values"][:, :, :, past:past + n] = s["values"][:, :, :, at]
    return {"keys": s["keys"], "values": s["values"]}


def _plain_thin(s):
    rows = s["rows"].long()
    s["to_keys"].copy_(s["keys"][:, :, rows])
    s["to_values"][..., :len(rows)] = s["values"][..., rows]
    return {"keys": s["to_keys"], "values": s["to_values"]}


# ------------------------------------------------- the library's own calls --

_ctx = None


def _context():
    """(the library's module, its context on the current device)."""
    global _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-inference-webgpu_amd"))
        import qwen_hip
        _ctx = (qwen_hip, qwen_hip.GpuContext.create(torch.cuda.current_device()))
    return _ctx


def _handles(s):
    """The state's tensors as the library's buffers, made once: they stay where they are."""
    if "buf" not in s:
        H, ctx = _context()
        b = s["buf"] = {n: H.DeviceBuffer(ctx, t.data_ptr(), t.numel() * t.element_size()) for n, t in s.items() if isinstance(t, torch.Tensor)}
        c = s["case"]
        if c["kind"] in ("commit", "thin"):
            lists = {"": s["keys"].shape[2], "to_": c.get("keep")}
            for to, cap in lists.items():
                if cap is not None:
                    b[to + "kv"] = ctx.kv_list(b[to + "keys"], b[to + "values"], cap, s[to + "keys"][0].numel(), s[to + "values"][0].numel())
    return s["buf"]


def _own(s):
    c, ctx, b = s["case"], _context()[1], _handles(s)
    k = c["kind"]
    if k == "append":
        cap = c["past"] + c["nodes"]
        ctx.rope_append_tree(b["q"], b["k"], b["v"], b["cos"], b["sin"], cap, b["depth"], b["qr"], b["keys"], b["values"], cap,
                             c["heads"], c["kv"], HD, c["past"], c["nodes"])
        return {"q": s["qr"], "keys": s["keys"], "values": s["values"]}
    if k == "attn":
        ctx.attention_tree(b["q"], b["keys"], b["values"], c["past"] + c["nodes"], b["mask"], b["out"], c["nodes"], c["past"],
                           c["heads"], c["kv"])
        return {"out": s["out"]}
    if k == "verify":
        ctx.verify_tree(b["logits"], b.get("draft"), b["tokens"], b["parent"], c["nodes"], c["vocab"], s["temperature"],
                        b["uniform"], b["path"], b["count"], b["next"])
        return {"path": s["path"], "count": s["count"], "next": s["next"]}
    if k == "commit":
        ctx.kv_gather(b["kv"], c["past"], b["kv"], c["past"], c["layers"], c["kv"], HD, b["rows"], c["nodes"], b["count"])
        return {"keys": s["keys"], "values": s["values"]}
    ctx.kv_gather(b["kv"], 0, b["to_kv"], 0, c["layers"], c["kv"], HD, b["rows"], c["keep"])
    return {"keys": s["to_keys"], "values": s["to_values"]}


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attn": _plain_attention, "verify": _plain_verify, "commit": _plain_commit, "thin": _plain_thin}[s["case"]["kind"]](s)


# ------------------------------------------------------ bytes and operations --

def work(case):
    k = case["kind"]
    if k == "append":
        n, h, kv = case["nodes"], case["heads"], case["kv"]
        return {"bytes": n * (8 * h * HD + 2 * kv * HD * 6 + 4 * HD + 4), "flops": 3 * n * (h + kv) * HD}
    if k == "attn":
        n, h, total = case["nodes"], case["heads"], case["past"] + case["nodes"]
        return {"bytes": 4 * case["kv"] * HD * total + 8 * n * h * HD + 8 * n * ((n + 63) // 64), "flops": 4 * n * total * h * HD}
    if k == "verify":
        # One root-to-leaf path: the walk needs no other node's rows.
        rows = case["depth"] + 1
        draft = case["depth"] if case["how"] == "sampled" else 0
        return {"bytes": 4 * case["vocab"] * (rows + draft) + 24 * case["nodes"], "flops": case["vocab"] * (3 * rows + 3 * draft)}
    rows = case["count"] - 1 if k == "commit" else case["keep"]
    return {"bytes": max(8 * case["layers"] * case["kv"] * HD * rows, 4) + 4 * rows, "flops": 0}


# ------------------------------------------------------------ f64 evaluation --

def exact(case, seed):
    s, k = prepare(case, seed), case["kind"]
    if k == "append":
        n, past = case["nodes"], case["past"]
        keys, values = s["keys"].double(), s["values"].double()
        q = s["q"].double().reshape(n, -1, 2, HD // 2)
        kk = s["k"].double().reshape(n, -1, 2, HD // 2)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[past + s["depth"].long()][:, None]
        q, kk = (torch.complex(t[:, :, 0], t[:, :, 1]) * turn for t in (q, kk))
        q, kk = (torch.cat((t.real, t.imag), 2) for t in (q, kk))
        keys[:, past:past + n] = kk.permute(1, 0, 2)
        values[:, :, past:past + n] = s["v"].double().reshape(n, -1, HD).permute(1, 2, 0)
        return {"q": q.reshape(n, -1), "keys": keys, "values": values}
    if k == "attn":
        n, past, kv, heads = case["nodes"], case["past"], case["kv"], case["heads"]
        see = torch.ones((n, past + n), dtype=torch.bool, device="cuda")
        bits = np.unpackbits(s["mask"].cpu().numpy().view(np.uint8).reshape(n, -1), axis=1, bitorder="little")[:, :n]
        see[:, past:] = torch.from_numpy(bits).cuda() != 0
        q = s["q"].double().reshape(n, heads, HD)
        out = torch.empty_like(q)
        for h in range(heads):
            g = h // (heads // kv)
            z = (q[:, h] @ s["keys"][g].double().T.contiguous()) / 8
            out[:, h] = torch.softmax(z.masked_fill(~see, -math.inf), 1) @ s["values"][g, :, :past + n].double().T.contiguous()
        return {"out": out.reshape(n, -1)}
    if k == "verify":
        return _exact_verify(s)
    if k == "commit":
        past, count = case["past"], case["count"]
        keys, values, rows = s["keys"].double(), s["values"].double(), s["rows"].cpu().tolist()
        old = keys[:, :, past:].clone(), values[..., past:].clone()
        for j in range(count):
            keys[:, :, past + j] = old[0][:, :, rows[j]]
            values[..., past + j] = old[1][..., rows[j]]
        return {"keys": keys, "values": values}
    rows, values = s["rows"].long(), s["to_values"].double()
    values[..., :len(rows)] = torch.index_select(s["values"], 3, rows).double()
    return {"keys": torch.index_select(s["keys"], 2, rows).double(), "values": values}


def _exact_verify(s):
    """The walk from the root, child by child, on the host."""
    n = s["case"]["nodes"]
    parent, tokens, u = (s[x].cpu().numpy() for x in ("parent", "tokens", "uniform"))
    path, at, dist = [0], 0, None

    def start(i):
        z = s["logits"][i].cpu().numpy().astype(np.float64)
        if s["temperature"] == 0:
            return (np.arange(len(z)) == np.argmax(z)).astype(np.float64)
        e = np.exp((z - z.max()) / s["temperature"])
        return e / e.sum()

    dist = start(0)
    for i in range(1, n):
        if parent[i] != at:
            continue
        x = tokens[i]
        if s["draft"] is not None:
            q = s["draft"][at].cpu().numpy().astype(np.float64)
        else:
            q = (np.arange(len(dist)) == x).astype(np.float64)
        if u[i] * q[x] < dist[x]:
            path.append(i)
            at, dist = i, start(i)
        elif s["temperature"] != 0:
            dist = np.maximum(dist - q, 0)
            dist /= dist.sum()
    nxt = int(np.argmax(dist)) if s["temperature"] == 0 else int(np.argmax((np.cumsum(dist) > u[0] * dist.sum()) & (dist > 0)))
    return {"path": np.array(path + [-1] * (n - len(path)), np.int32), "count": np.array([len(path)], np.int32),
            "next": np.array([nxt], np.int32)}
