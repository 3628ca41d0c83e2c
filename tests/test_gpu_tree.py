"""Decoding from a tree of drafts on the GPU: each operator against its 64-bit restatement
(tree_lib.py), at the sizes, masks and values where it can go wrong, and a run of them together
against a decode token by token."""
import ctypes
import threading

import numpy as np
import pytest

import tree_lib as T

pytestmark = pytest.mark.gpu

NAN16 = 0x7E00


def _vstride(cap):
    return (cap + 63) // 64 * 64


def _f16(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def _caches(rng, kv, cap, used):
    """Random caches of `used` positions; what lies behind them is NaN."""
    keys, values = _f16(rng, kv, cap, 64), np.full((kv, 64, _vstride(cap)), np.nan, np.float16)
    keys[:, used:] = np.nan
    values[..., :used] = _f16(rng, kv, 64, used)
    return keys, values


# ---------------------------------------------------------------- attention --

def _attend(ctx, q, keys, values, mask, past, heads, kv):
    n, cap = q.shape[0], keys.shape[1]
    bufs = [ctx.upload(x) for x in (q, keys, values, mask)]
    out = ctx.upload(np.full((n, heads * 64), np.nan, np.float32))
    ctx.attention_tree(bufs[0], bufs[1], bufs[2], cap, bufs[3], out, n, past, heads, kv)
    got = out.read().reshape(n, heads, 64)
    for b in bufs + [out]:
        b.free()
    return got


def _check_attention(ctx, q, keys, values, see, past, heads, kv, mask=None, rms=1e-6):
    got = _attend(ctx, q, keys, values, T.pack(see) if mask is None else mask, past, heads, kv)
    want, size, reach = T.attention(q.reshape(-1, heads, 64), keys, values, see, past, heads // kv)
    # A score is off by at most 64 f32 roundings of its products' sum and the 2^-20 of q's two f16
    # terms and its scale; a weight by that much in the exponent, both above and below the line,
    # and 2^-20 of its own terms; each of the P sums of the output by 2^-24 of their size.
    total = past + q.shape[0]
    tol = size * (2 * reach * (64 * 2.0**-24 + 2.0**-20) + 2.0**-20 + (total + 64) * 2.0**-24) + 1e-30
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])
    if np.abs(want).max() > 0:  # what the header states of the output
        assert np.linalg.norm(got - want) <= rms * np.linalg.norm(want)
    return got


SHAPES = [(1, 0, 14, 2), (1, 1, 14, 2), (1, 127, 2, 1), (2, 63, 4, 4), (5, 123, 14, 2), (7, 57, 1, 1), (9, 64, 9, 3),
          (16, 1024, 14, 2), (17, 31, 32, 2), (33, 0, 14, 2), (63, 500, 14, 2), (64, 1000, 4, 2), (65, 129, 14, 2), (100, 40, 7, 7),
          (130, 2000, 14, 1), (200, 3, 4, 2), (3, 9000, 14, 2), (12, 500, 14, 2), (11, 513, 3, 3), (48, 3333, 14, 2),
          # long enough and wide enough for the shared stages
          (300, 6000, 20, 4), (700, 1900, 16, 1), (64, 32700, 14, 2), (65, 12863, 32, 1)]


@pytest.mark.parametrize("nodes,past,heads,kv", SHAPES)
def test_attention_of_a_tree(ctx, nodes, past, heads, kv):
    rng = np.random.default_rng(nodes * 131 + past)
    keys, values = _caches(rng, kv, past + nodes + int(rng.integers(0, 70)), past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    _, see = T.plan(T.random_tree(rng, nodes))
    _check_attention(ctx, q, keys, values, see, past, heads, kv)


@pytest.mark.parametrize("nodes,past,heads,kv", [(1, 0, 2, 1), (5, 0, 14, 2), (40, 0, 14, 2), (70, 33, 4, 2), (129, 0, 2, 2),
                                                    (600, 0, 2, 2), (1300, 0, 32, 1)])
def test_attention_of_any_mask(ctx, nodes, past, heads, kv):
    """Random bits, rows that see nothing, bits behind the last node."""
    rng = np.random.default_rng(nodes + past)
    keys, values = _caches(rng, kv, past + nodes, past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    see = rng.random((nodes, nodes)) < 0.3
    see[::3] = False
    see[nodes // 2] = True
    see[0] = False
    mask = T.pack(see)
    if nodes % 64:
        mask[:, -1] |= np.uint64(2**64 - 2**(nodes % 64))
    got = _check_attention(ctx, q, keys, values, see, past, heads, kv, mask)
    if past == 0:
        assert not got[0].any()


@pytest.mark.parametrize("nodes,past,heads,kv", [(6, 20, 14, 2), (40, 70, 4, 2), (96, 10, 14, 2), (17, 3000, 14, 2),
                                                    (64, 12900, 32, 1)])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_attention_is_untouched_by_what_a_node_does_not_see(ctx, nodes, past, heads, kv, what):
    """Infinities and NaN in the K and V rows of hidden nodes change no bit; a node that sees an
    infinite value gets it."""
    rng = np.random.default_rng(nodes)
    keys, values = _caches(rng, kv, past + nodes, past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    _, see = T.plan(T.random_tree(rng, nodes))
    hidden = [nodes // 2, nodes - 1]
    see[:, hidden] = False
    want = _attend(ctx, q, keys, values, T.pack(see), past, heads, kv)
    assert np.isfinite(want).all()
    keys[:, past + np.array(hidden)] = what
    values[:, ::2, past + np.array(hidden)] = what
    values[:, 1, past + hidden[0]] = what
    got = _attend(ctx, q, keys, values, T.pack(see), past, heads, kv)
    np.testing.assert_array_equal(got, want)
    # Now one node sees one of them, whose key is finite: only its outputs change, to what the value says.
    keys[:, past + hidden[0]] = _f16(rng, kv, 64)
    see[1, hidden[0]] = True
    got = _attend(ctx, q, keys, values, T.pack(see), past, heads, kv)
    rest = np.arange(nodes) != 1
    np.testing.assert_array_equal(got[rest], want[rest])
    touched = np.array([d % 2 == 0 or d == 1 for d in range(64)])
    assert (np.isnan(got[1][:, touched]).all() if np.isnan(what) else (got[1][:, touched] == what).all())
    assert np.isfinite(got[1][:, ~touched]).all()


@pytest.mark.parametrize("nodes,past,heads,kv", [(6, 20, 14, 2), (20, 3000, 14, 2), (64, 12900, 32, 1)])
def test_attention_adds_the_infinite_values_that_a_node_sees(ctx, nodes, past, heads, kv):
    """Infinities of both signs in a dimension are NaN, of one sign that infinity, with a NaN before past NaN."""
    rng = np.random.default_rng(nodes)
    keys, values = _caches(rng, kv, past + nodes, past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    _, see = T.plan(T.random_tree(rng, nodes))
    see[-1] = False
    see[-1, [1, 2, nodes - 1]] = True
    see[:-1, [1, 2]] = False
    want = _attend(ctx, q, keys, values, T.pack(see), past, heads, kv)
    values[:, 3, past + 1] = np.inf
    values[:, 4, past + 1], values[:, 4, past + 2] = np.inf, -np.inf
    values[:, 5, past + 2] = -np.inf
    values[:, 6, past + 1], values[:, 6, past // 2] = np.inf, np.nan
    got = _attend(ctx, q, keys, values, T.pack(see), past, heads, kv)
    assert (got[-1][:, 3] == np.inf).all() and (got[-1][:, 5] == -np.inf).all()
    assert np.isnan(got[-1][:, 4]).all() and np.isnan(got[:, :, 6]).all()
    same = np.ones(want.shape, bool)
    same[-1, :, 3:6] = same[:, :, 6] = False
    np.testing.assert_array_equal(got[same], want[same])


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 30.0, 1e4])
def test_attention_of_small_and_large_queries(ctx, scale):
    """Scores from next to nothing to ones that leave a single weight: q is no f16 number."""
    rng = np.random.default_rng(3)
    nodes, past, heads, kv = 12, 300, 14, 2
    keys, values = _caches(rng, kv, past + nodes, past + nodes)
    q = (rng.standard_normal((nodes, heads * 64)) * scale).astype(np.float32)
    _, see = T.plan(T.random_tree(rng, nodes))
    _check_attention(ctx, q, keys, values, see, past, heads, kv, rms=1e-6 * max(1.0, scale))


def test_attention_where_one_weight_leads_many_small_ones(ctx):
    """One key scores 17 above thousands of others, whose weights of 4e-8 still sum to 1e-4."""
    rng = np.random.default_rng(8)
    nodes, past = 4, 4000
    keys, values = np.zeros((1, past + nodes, 64), np.float16), np.zeros((1, 64, _vstride(past + nodes)), np.float16)
    q = np.zeros((nodes, 64), np.float32)
    q[:, 0] = 17 * 8
    keys[0, 5, 0] = 1
    values[0, :, :past + nodes] = 1 + rng.random((64, past + nodes)).astype(np.float16)
    values[0, :, 5] = 0
    _, see = T.plan(np.array([-1, 0, 1, 0], np.int32))
    _check_attention(ctx, q, keys, values, see, past, 1, 1, rms=1e-4)


def test_attention_of_a_chain_is_causal_attention(ctx):
    rng = np.random.default_rng(4)
    nodes, past, heads, kv = 9, 700, 14, 2
    keys, values = _caches(rng, kv, past + nodes, past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    got = _attend(ctx, q, keys, values, T.pack(np.tril(np.ones((nodes, nodes), bool))), past, heads, kv)
    bufs, out = [ctx.upload(x) for x in (q, keys, values)], ctx.empty(q.nbytes)
    ctx.attention(*bufs, past + nodes, out, nodes, past, heads, kv, kind="exact")
    want = out.read().reshape(nodes, heads, 64)
    assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want)  # two f32 evaluations, 1e-6 each


@pytest.mark.parametrize("nodes,past,heads,kv", [(3, 20, 14, 2), (17, 1500, 9, 3), (64, 12900, 32, 1)])
def test_attention_writes_its_rows_alone(ctx, nodes, past, heads, kv):
    """What lies before and behind out, the queries, the mask and the caches keep their bits."""
    rng = np.random.default_rng(nodes)
    keys, values = _caches(rng, kv, past + nodes + 5, past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    mask = T.pack(T.plan(T.random_tree(rng, nodes))[1])
    room = np.full(q.size + 128, 7.25, np.float32)
    given = (q, keys, values, mask)
    bufs, out = [ctx.upload(x) for x in given], ctx.upload(room)
    inner = type(out)(ctx, out.ptr + 256, q.nbytes)
    ctx.attention_tree(bufs[0], bufs[1], bufs[2], past + nodes + 5, bufs[3], inner, nodes, past, heads, kv)
    got = out.read()
    assert (got[:64] == 7.25).all() and (got[-64:] == 7.25).all() and (got[64:-64] != 7.25).all()
    for b, x in zip(bufs, given):
        np.testing.assert_array_equal(b.read(np.uint8), np.frombuffer(np.ascontiguousarray(x).tobytes(), np.uint8))


def test_attention_behind_four_billion_bytes(ctx):
    """A cache whose last kv head starts behind 2^32 bytes and 2^31 values."""
    rng = np.random.default_rng(6)
    nodes, past, heads, kv, cap = 5, 70, 8, 4, 12_000_000
    keys, values = ctx.empty(kv * cap * 128), ctx.empty(kv * 64 * _vstride(cap) * 2)
    k, v = _f16(rng, kv, past + nodes, 64), _f16(rng, kv, 64, past + nodes)

    def put(buf, offset, a):
        a = np.ascontiguousarray(a)
        assert ctx.lib.qh_upload(ctx.handle, buf.ptr + offset, a.ctypes.data, a.nbytes) == 0

    for h in range(kv):
        put(keys, h * cap * 128, k[h])
        for d in range(64):
            put(values, (h * 64 + d) * _vstride(cap) * 2, v[h, d])
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    _, see = T.plan(T.random_tree(rng, nodes))
    qb, mb, out = ctx.upload(q), ctx.upload(T.pack(see)), ctx.empty(q.nbytes)
    ctx.attention_tree(qb, keys, values, cap, mb, out, nodes, past, heads, kv)
    got = out.read().reshape(nodes, heads, 64)
    want, _, _ = T.attention(q.reshape(nodes, heads, 64), k, v, see, past, heads // kv)
    keys.free()
    values.free()
    assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


# ------------------------------------------------------------ rotate + append --

@pytest.mark.parametrize("nodes,past,heads,kv,hd", [(1, 0, 14, 2, 64), (5, 123, 14, 2, 64), (64, 1000, 14, 2, 64), (130, 7, 4, 4, 64),
                                                    (3, 5, 3, 1, 2), (7, 9, 4, 2, 30), (66, 61, 8, 1, 128)])
def test_rope_append_tree(ctx, hip, nodes, past, heads, kv, hd):
    rng = np.random.default_rng(nodes + hd)
    cap = past + nodes + 9
    q, k, v = (rng.standard_normal((nodes, h, hd)).astype(np.float32) for h in (heads, kv, kv))
    depth = rng.integers(0, nodes, nodes).astype(np.int32)
    cos, sin = hip.rope_tables(hd, 1e6, past + nodes)
    keys, values = _f16(rng, kv, cap, hd), _f16(rng, kv, hd, _vstride(cap))
    given = depth.copy()
    if nodes > 2:
        given[1], given[2] = -5, nodes + 3
        depth[1], depth[2] = 0, nodes - 1
    b = {n: ctx.upload(x) for n, x in dict(q=q, k=k, v=v, cos=cos, sin=sin, depth=given, kc=keys, vc=values).items()}
    out = ctx.empty(q.nbytes)
    ctx.rope_append_tree(b["q"], b["k"], b["v"], b["cos"], b["sin"], past + nodes, b["depth"], out, b["kc"], b["vc"], cap, heads,
                         kv, hd, past, nodes)
    c, s = (t[past + depth][:, None].astype(np.float64) for t in (cos, sin))
    half = hd // 2

    def rot(x):
        lo, hi = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
        return np.concatenate((lo * c - hi * s, hi * c + lo * s), 2), np.concatenate((abs(lo * c) + abs(hi * s), abs(hi * c) + abs(lo * s)), 2)

    # two products and their sum, each rounded to f32
    want, size = rot(q)
    got = out.read().reshape(q.shape)
    assert (np.abs(got - want) <= 2 * 2.0**-24 * size + 1e-30).all()
    np.testing.assert_array_equal(b["q"].read().reshape(q.shape), q)
    want, size = rot(k)
    gk, gv = b["kc"].read(np.float16).reshape(keys.shape), b["vc"].read(np.float16).reshape(values.shape)
    new = gk[:, past:past + nodes].astype(np.float64)
    # the f32 value's error, then half an f16 step
    assert (np.abs(new - want.transpose(1, 0, 2)) <= (2 * 2.0**-24 * size + np.abs(want) * 2.0**-11 + 2.0**-25).transpose(1, 0, 2)).all()
    keys[:, past:past + nodes] = gk[:, past:past + nodes]
    values[..., past:past + nodes] = v.astype(np.float16).transpose(1, 2, 0)
    np.testing.assert_array_equal(gk, keys)
    np.testing.assert_array_equal(gv, values)


def test_rope_append_of_a_chain_is_rope_and_append(ctx, hip):
    """Bit for bit qh_rope and qh_kv_append, with q rotated where it lies."""
    rng = np.random.default_rng(2)
    nodes, past, heads, kv, cap = 21, 40, 14, 2, 70
    q, k, v = (rng.standard_normal((nodes, h * 64)).astype(np.float32) for h in (heads, kv, kv))
    cos, sin = (ctx.upload(t) for t in hip.rope_tables(64, 1e6, cap))
    empty = np.zeros((kv, cap, 64), np.float16), np.zeros((kv, 64, _vstride(cap)), np.float16)
    a = [ctx.upload(x) for x in (q, k, v) + empty]
    b = [ctx.upload(x) for x in (q, k, v) + empty]
    depth = ctx.upload(np.arange(nodes, dtype=np.int32))
    ctx.rope_append_tree(*a[:3], cos, sin, cap, depth, a[0], a[3], a[4], cap, heads, kv, 64, past, nodes)
    ctx.rope(b[0], cos, sin, cap, nodes, heads, 64, past)
    ctx.rope(b[1], cos, sin, cap, nodes, kv, 64, past)
    ctx.kv_append(b[1], b[2], b[3], b[4], cap, kv, 64, past, nodes)
    np.testing.assert_array_equal(a[1].read().reshape(k.shape), k)
    for i in (0, 3, 4):
        np.testing.assert_array_equal(a[i].read(np.uint16), b[i].read(np.uint16))


# ------------------------------------------------------------- verification --

def _verify(ctx, logits, draft, tokens, parent, temperature, uniform):
    n, vocab = logits.shape
    bufs = [None if x is None else ctx.upload(x) for x in (logits, draft, tokens, parent, uniform)]
    path, count, nxt = (ctx.upload(np.full(m, 77, np.int32)) for m in (n + 3, 2, 2))
    ctx.verify_tree(bufs[0], bufs[1], bufs[2], bufs[3], n, vocab, temperature, bufs[4], path, count, nxt)
    p, c, t = path.read(), count.read(), nxt.read()
    assert (p[n:] == 77).all() and c[1] == 77 and t[1] == 77
    for b in bufs + [path, count, nxt]:
        if b is not None:
            b.free()
    assert (p[c[0]:n] == -1).all()
    return [int(x) for x in p[:c[0]]], int(t[0])


def _drafts(rng, nodes, vocab, how, width=3, std=2.5):
    parent = T.random_tree(rng, nodes, width)
    logits = (rng.standard_normal((nodes, vocab)) * std).astype(np.float32)
    noisy = logits + rng.standard_normal((nodes, vocab)).astype(np.float32) * 0.7
    q = np.exp(noisy - noisy.max(1, keepdims=True))
    q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    tokens = np.zeros(nodes, np.int32)
    for i in range(1, nodes):
        row = q[parent[i]].astype(np.float64)
        tokens[i] = rng.choice(vocab, p=row / row.sum())
        if how != "sampled" and rng.random() < 0.6:
            tokens[i] = logits[parent[i]].argmax()
    return logits, q if how == "sampled" else None, tokens, parent, rng.random(nodes)


@pytest.mark.parametrize("how", ["greedy", "lookup", "sampled"])
@pytest.mark.parametrize("nodes,vocab", [(1, 1), (1, 151936), (2, 2), (5, 63), (9, 1000), (33, 257), (6, 4096), (6, 4097), (70, 5000), (1024, 130), (3, 300001),
                                         (4, 40961), (12, 151936)])
def test_verify_tree(ctx, how, nodes, vocab):
    """Path and next token are the walk's, over several draws (f64 on both sides: a pick differs
    only where a random number lies within 1e-13 of a border)."""
    for seed in range(12 if vocab < 10000 else 4):
        rng = np.random.default_rng(nodes * 1000 + vocab + seed)
        logits, q, tokens, parent, u = _drafts(rng, nodes, vocab, how, width=1 + seed % 4)
        t = 0.0 if how == "greedy" else (1.0, 0.7, 0.2)[seed % 3]
        got = _verify(ctx, logits, q, tokens, parent, t, None if how == "greedy" else u)
        assert got == T.verify(logits, q, tokens, parent, t, u), (seed, t)


@pytest.mark.parametrize("how", ["greedy", "lookup", "sampled"])
def test_verify_tree_of_odd_values(ctx, how):
    """Masked, infinite and missing logits, equal logits, tokens twice among siblings and outside the
    vocabulary, parents that are none, random numbers at and beyond their ends, drafts without weight."""
    nodes, vocab = 24, 300
    for seed in range(40):
        rng = np.random.default_rng(seed)
        logits, q, tokens, parent, u = _drafts(rng, nodes, vocab, how, width=4)
        kind = seed % 8
        if kind == 0:
            logits[:, rng.random(vocab) < 0.7] = -np.inf
        elif kind == 1:
            logits[rng.random(logits.shape) < 0.2] = np.nan
            logits[:, 0] = np.where(rng.random(nodes) < 0.5, np.nan, logits[:, 0])
        elif kind == 2:
            logits[rng.random(logits.shape) < 0.02] = np.inf
        elif kind == 3:
            logits[rng.random(nodes) < 0.5] = -np.inf
            logits[0] = np.nan if seed % 16 == 3 else -np.inf
        elif kind == 4:
            logits = np.round(logits)
            tokens[1:] = logits[np.maximum(parent[1:], 0)].argmax(1)
            tokens[2::3] = tokens[1]
        elif kind == 5:
            tokens[rng.random(nodes) < 0.3] = rng.choice([-1, vocab, 2**31 - 1, -2**31])
            parent[rng.random(nodes) < 0.2] = rng.choice([-1, nodes, -2**31, 2**31 - 1, nodes - 1])
        elif kind == 6:
            u[:] = rng.choice([0.0, 1 - 2.0**-53, 1.0, 7.0, -1.0, np.nan], nodes)
        elif kind == 7 and q is not None:
            q[rng.random(q.shape) < 0.4] = 0
            q[rng.random(q.shape) < 0.1] = rng.choice([-1.0, np.nan, np.inf])
            q[0] *= 3
        t = 0.0 if how == "greedy" else 0.8
        late = parent >= np.arange(nodes)  # a parent that is no earlier node
        ref_parent = np.where(late | (parent < 0), -7, parent)
        got = _verify(ctx, logits, q, tokens, parent, t, u)
        assert got == T.verify(logits, q, tokens, ref_parent, t, u), (seed, kind)


def test_verify_tree_with_nothing_left(ctx):
    """All of p on the rejected tokens, drafts that cover more than p: the walk falls back on p."""
    vocab = 5000
    logits = np.full((3, vocab), -np.inf, np.float32)
    logits[:, [7, 4100]] = 0, np.log(3)
    parent, tokens = np.array([-1, 0, 0], np.int32), np.array([0, 7, 4100], np.int32)
    u = np.array([0.9, 0.3, 1.5])
    assert _verify(ctx, logits, None, tokens, parent, 1.0, u) == T.verify(logits, None, tokens, parent, 1.0, u) == ([0], 4100)
    draft = np.full((3, vocab), 2.0, np.float32)
    u = np.array([0.1, 0.999, 0.999])
    assert _verify(ctx, logits, draft, tokens, parent, 1.0, u) == T.verify(logits, draft, tokens, parent, 1.0, u) == ([0], 7)


@pytest.mark.parametrize("how", ["lookup", "sampled"])
@pytest.mark.parametrize("temperature", [1e-30, 1e-9, 1e-3, 1e3, 1e30])
def test_verify_tree_of_any_scale(ctx, how, temperature):
    """Logits from the temperature's size to 2^30 and more times it, some masked by the lowest f32, chunks of those alone."""
    vocab, nodes = 9000, 9
    for seed, scale in enumerate((1.0, 30.0, 1e4, 2.0**29, 2.0**31, 1e12)):
        rng = np.random.default_rng(seed)
        logits, q, tokens, parent, u = _drafts(rng, nodes, vocab, how)
        top = min(temperature * scale, 1e37)
        logits = np.clip(logits * np.float64(temperature) - top * rng.integers(0, 2, (nodes, 1)), -3e38, 3e38).astype(np.float32)
        logits[rng.random(logits.shape) < 0.3] = np.finfo(np.float32).min
        logits[seed % nodes, 4096:8192] = np.finfo(np.float32).min
        for i in range(1, nodes, 2):
            tokens[i] = logits[parent[i]].argmax()
        assert _verify(ctx, logits, q, tokens, parent, temperature, u) == T.verify(logits, q, tokens, parent, temperature, u), scale


@pytest.mark.parametrize("how", ["greedy", "lookup", "sampled"])
@pytest.mark.parametrize("nodes,vocab", [(14, 9001), (64, 4100), (200, 9000)])
def test_verify_tree_of_one_generation(ctx, how, nodes, vocab):
    """All drafts under the root, some of them twice, with random numbers that reject most: more rejections than
    have launches of their own, a draw from what they left."""
    for seed in range(6):
        rng = np.random.default_rng(seed)
        logits, q, tokens, parent, u = _drafts(rng, nodes, vocab, how)
        parent[1:] = 0
        tokens[1:] = rng.choice(vocab, nodes - 1, p=(e := np.exp(logits[0].astype(np.float64))) / e.sum())
        u[1:] = 1 - u[1:] * (0.02 if seed % 2 else 0.2)
        t = 0.0 if how == "greedy" else 0.9
        assert _verify(ctx, logits, q, tokens, parent, t, u) == T.verify(logits, q, tokens, parent, t, u), seed


@pytest.mark.parametrize("how", ["greedy", "lookup", "sampled"])
def test_verify_tree_of_the_largest_vocabulary(ctx, how):
    vocab = 1 << 24
    rng = np.random.default_rng(11)
    logits = rng.standard_normal((3, vocab), np.float32) * np.float32(2.5)
    draft = None
    if how == "sampled":
        draft = np.exp(logits[:, ::-1]) / np.float32(4e8)  # of other tokens than the target's
    parent, tokens = np.array([-1, 0, 0], np.int32), np.array([0, int(logits[0].argmin()), vocab - 1], np.int32)
    for u in (np.array([0.3, 0.99, 0.9]), np.array([0.97, 0.99, 0.0]), np.array([1 - 2.0**-53, 0.99, 0.99])):
        t = 0.0 if how == "greedy" else 0.7
        assert _verify(ctx, logits, draft, tokens, parent, t, u) == T.verify(logits, draft, tokens, parent, t, u)


# ------------------------------------------------------------------- gather --

def _kv(rng, layers, kv, hd, cap, pad=0):
    """Bit patterns of `layers` caches with `pad` values between them."""
    k = rng.integers(0, 65536, (layers, kv * cap * hd + pad)).astype(np.uint16)
    v = rng.integers(0, 65536, (layers, kv * hd * _vstride(cap) + pad)).astype(np.uint16)
    return k, v


def _gather(ctx, src, src_cap, src_base, dst, dst_cap, dst_base, layers, kv, hd, rows, n, count):
    """The caches after the call, src is dst for a call in place; checks that nothing else moved."""
    same = src is dst
    bufs = [ctx.upload(x) for x in src] + ([] if same else [ctx.upload(x) for x in dst])
    a = ctx.kv_list(bufs[0], bufs[1], src_cap, src[0].shape[1], src[1].shape[1])
    b = a if same else ctx.kv_list(bufs[2], bufs[3], dst_cap, dst[0].shape[1], dst[1].shape[1])
    ctx.kv_gather(a, src_base, b, dst_base, layers, kv, hd, None if rows is None else ctx.upload(rows), n,
                  None if count is None else ctx.upload(np.array([count], np.int32)))
    got = [x.read(np.uint16).reshape(y.shape) for x, y in zip(bufs[-2:], dst)]

    def split(c, cap):
        ke, ve = kv * cap * hd, kv * hd * _vstride(cap)
        return (c[0][:, :ke].reshape(layers, kv, cap, hd), c[1][:, :ve].reshape(layers, kv, hd, -1)), (c[0][:, ke:], c[1][:, ve:])

    (sk, sv), _ = split(src, src_cap)
    (dk, dv), gap = split(dst, dst_cap)
    (gk, gv), got_gap = split(got, dst_cap)
    want_k, want_v = T.gather(sk, sv, src_base, dk, dv, dst_base, rows, n, count, same)
    np.testing.assert_array_equal(gk, want_k)
    np.testing.assert_array_equal(gv, want_v)
    for x, y in zip(gap, got_gap):
        np.testing.assert_array_equal(x, y)
    if not same:
        for x, y in zip(src, bufs[:2]):
            np.testing.assert_array_equal(y.read(np.uint16).reshape(x.shape), x)


@pytest.mark.parametrize("layers,kv,hd,cap,base,rows", [
    (1, 1, 64, 8, 0, [0]), (3, 2, 64, 40, 30, [0, 2, 3, 7]), (24, 2, 64, 133, 70, [0, 1, 5, 20, 62]),
    (2, 2, 64, 700, 5, "thin"), (1, 3, 8, 4000, 0, "thin"), (2, 1, 128, 513, 1, "thin"), (1, 2, 24, 70, 3, [4, 3, 2, 1, 0, 5, 9, 9])])
def test_gather_in_place(ctx, layers, kv, hd, cap, base, rows):
    rng = np.random.default_rng(cap)
    if rows == "thin":
        rows = np.sort(rng.choice(cap - base, (cap - base) * 2 // 3, replace=False))
    rows = np.array(rows, np.int32)
    for count in (None, len(rows), len(rows) // 2, 0, -3, len(rows) + 5):
        c = _kv(rng, layers, kv, hd, cap, pad=16 if count else 0)
        _gather(ctx, c, cap, base, c, cap, base, layers, kv, hd, rows, len(rows), count)
    # rows from further on, moved to the front; then rows that are none
    c = _kv(rng, layers, kv, hd, cap)
    n = min(len(rows), cap - base)
    _gather(ctx, c, cap, min(base + 3, cap - 1), c, cap, 0, layers, kv, hd, rows[:n], n, None)
    odd = rows[:n].copy()
    odd[::2] = rng.choice([-1, cap, 2**31 - 1, -2**31], len(odd[::2]))
    _gather(ctx, c, cap, base, c, cap, base, layers, kv, hd, odd, n, None)


@pytest.mark.parametrize("layers,kv,hd,src_cap,dst_cap,n", [(1, 1, 64, 1, 1, 1), (24, 2, 64, 100, 64, 33), (2, 3, 64, 1000, 1111, 777),
                                                            (3, 1, 8, 70, 65, 65), (1, 2, 128, 5000, 2048, 2000), (2, 2, 40, 129, 513, 300)])
def test_gather_between_caches(ctx, layers, kv, hd, src_cap, dst_cap, n):
    rng = np.random.default_rng(src_cap + n)
    src, dst = _kv(rng, layers, kv, hd, src_cap, 8), _kv(rng, layers, kv, hd, dst_cap, 24)
    rows = rng.integers(0, src_cap, n).astype(np.int32)  # any order, some twice
    _gather(ctx, src, src_cap, 0, dst, dst_cap, 0, layers, kv, hd, rows, n, None)
    rows = np.sort(rows)
    rows[::7] = -1
    _gather(ctx, src, src_cap, src_cap // 3, dst, dst_cap, dst_cap - n, layers, kv, hd, rows, n, n - n // 3)
    n = min(n, src_cap)
    for sb, db in ((0, 0), (src_cap - n, dst_cap - n)):  # a copy as it is
        _gather(ctx, src, src_cap, sb, dst, dst_cap, db, layers, kv, hd, None, n, None)


def test_gather_of_wide_heads(ctx):
    """The widest head, with rows over several steps of a block."""
    rng = np.random.default_rng(1)
    c = _kv(rng, 2, 2, 1024, 150, 8)
    rows = np.sort(rng.choice(140, 90, replace=False)).astype(np.int32)
    _gather(ctx, c, 150, 9, c, 150, 9, 2, 2, 1024, rows, 90, None)
    _gather(ctx, c, 150, 0, _kv(rng, 2, 2, 1024, 91), 91, 1, 2, 2, 1024, rows, 90, 77)


def test_append_and_gather_behind_four_billion_bytes(ctx):
    """The last kv head's rows start behind 2^32 bytes and 2^31 values, the tables' rows behind 2^30 bytes."""
    rng = np.random.default_rng(7)
    nodes, heads, kv, cap = 6, 8, 4, 12_000_000
    past = cap - 70
    keys, values, cos, sin = (ctx.empty(b) for b in (kv * cap * 128, kv * 64 * _vstride(cap) * 2, cap * 128, cap * 128))
    q, k, v = (rng.standard_normal((nodes, h * 64)).astype(np.float32) for h in (heads, kv, kv))
    depth = np.array([0, 1, 1, 2, 3, 2], np.int32)
    angle = rng.standard_normal((nodes, 32))

    def piece(call, buf, offset, a):
        assert call(ctx.handle, *((a.ctypes.data, buf.ptr + offset) if call is ctx.lib.qh_download else
                                  (buf.ptr + offset, a.ctypes.data)), a.nbytes) == 0
        return a

    for t, f in ((cos, np.cos), (sin, np.sin)):
        piece(ctx.lib.qh_upload, t, past * 128, f(angle).astype(np.float32))
    bufs = [ctx.upload(x) for x in (q, k, v, depth, np.array([0, 1, 3, 5], np.int32))]
    out = ctx.empty(q.nbytes)
    ctx.rope_append_tree(*bufs[:3], cos, sin, cap, bufs[3], out, keys, values, cap, heads, kv, 64, past, nodes)

    def rows(n):
        return (np.stack([piece(ctx.lib.qh_download, keys, (h * cap + past) * 128, np.empty((n, 64), np.float16)) for h in range(kv)]),
                np.stack([[piece(ctx.lib.qh_download, values, ((h * 64 + d) * _vstride(cap) + past) * 2, np.empty(n, np.float16))
                           for d in range(64)] for h in range(kv)]))

    got_k, got_v = rows(nodes)
    np.testing.assert_array_equal(got_v, v.reshape(nodes, kv, 64).transpose(1, 2, 0).astype(np.float16))
    x = k.reshape(nodes, kv, 2, 32).astype(np.float64)
    turn = np.exp(1j * angle)[depth][:, None]
    want = (x[:, :, 0] + 1j * x[:, :, 1]) * turn
    want = np.concatenate((want.real, want.imag), 2).transpose(1, 0, 2)
    # the tables' and the products' roundings to f32 of values below 8, then half an f16 step
    assert (np.abs(got_k - want) <= 6 * 2.0**-24 * 8 + np.abs(want) * 2.0**-11 + 2.0**-25).all()
    c = ctx.kv_list(keys, values, cap)
    ctx.kv_gather(c, past, c, past, 1, kv, 64, bufs[4], 4, None)
    new_k, new_v = rows(nodes)
    take = [0, 1, 3, 5, 4, 5]  # what lies behind the four stays
    np.testing.assert_array_equal(new_k, got_k[:, take])
    np.testing.assert_array_equal(new_v, got_v[..., take])
    for b in (keys, values, cos, sin):
        b.free()


# -------------------------------------------------------------- all together --

class _Small:
    """A two-layer model made of the library's operators: attention over the caches, residuals, a head."""

    heads, kv, vocab, layers, cap = 4, 2, 512, 2, 200

    def __init__(self, ctx, hip, seed):
        rng = np.random.default_rng(seed)
        self.ctx, self.hip, self.d = ctx, hip, self.heads * 64
        self.embed = rng.standard_normal((self.vocab, self.d)).astype(np.float32)
        self.keep = []

        def matrix(rows, std):
            b = ctx.upload((rng.standard_normal((rows, self.d)) * std).astype(np.float16).view(np.uint16))
            self.keep.append(b)
            return ctx.weight(hip.FMT_F16, rows, self.d, b)

        s = self.d ** -0.5
        self.w = [[matrix(r, 2 * s) for r in (self.d, self.kv * 64, self.kv * 64)] for _ in range(self.layers)]
        self.head = matrix(self.vocab, 3 * s)
        self.cos, self.sin = (ctx.upload(t) for t in hip.rope_tables(64, 1e4, self.cap))
        self.kel, self.vel = self.kv * self.cap * 64, self.kv * 64 * _vstride(self.cap)

    def caches(self):
        return (self.ctx.upload(np.zeros((self.layers, self.kel), np.float16)),
                self.ctx.upload(np.zeros((self.layers, self.vel), np.float16)))

    def at(self, cache, layer):
        k, v = cache
        D = self.hip.DeviceBuffer
        return D(self.ctx, k.ptr + 2 * layer * self.kel, 2 * self.kel), D(self.ctx, v.ptr + 2 * layer * self.vel, 2 * self.vel)

    def forward(self, tokens, cache, past, tree=None):
        """Logits [n, vocab] on the device; tree: (depth, mask) buffers, else a chain by the older operators."""
        ctx, n = self.ctx, len(tokens)
        x = ctx.upload(self.embed[np.asarray(tokens)])
        q, o = ctx.empty(x.nbytes), ctx.empty(x.nbytes)
        k, v = (ctx.empty(n * self.kv * 64 * 4) for _ in range(2))
        for i, (wq, wk, wv) in enumerate(self.w):
            kc, vc = self.at(cache, i)
            for w, y in ((wq, q), (wk, k), (wv, v)):
                ctx.matvec(w, x, None, y, n)
            if tree:
                ctx.rope_append_tree(q, k, v, self.cos, self.sin, self.cap, tree[0], q, kc, vc, self.cap, self.heads, self.kv,
                                     64, past, n)
                ctx.attention_tree(q, kc, vc, self.cap, tree[1], o, n, past, self.heads, self.kv)
            else:
                ctx.rope(q, self.cos, self.sin, self.cap, n, self.heads, 64, past)
                ctx.rope(k, self.cos, self.sin, self.cap, n, self.kv, 64, past)
                ctx.kv_append(k, v, kc, vc, self.cap, self.kv, 64, past, n)
                ctx.attention(q, kc, vc, self.cap, o, n, past, self.heads, self.kv)
            ctx.add(x, o, n * self.d)
        logits = ctx.empty(n * self.vocab * 4)
        ctx.matvec(self.head, x, None, logits, n)
        return logits


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_decoding_from_trees_is_decoding_token_by_token(ctx, hip, seed):
    """Greedy decoding: trees that hold some of the true continuation among wrong drafts give the
    tokens and the cache of a decode token by token."""
    m, rng = _Small(ctx, hip, seed), np.random.default_rng(seed)
    prompt = rng.integers(0, m.vocab, 9)
    slow = m.caches()
    m.forward(prompt[:-1], slow, 0)
    truth = [int(prompt[-1])]
    for i in range(40):
        row = m.forward(truth[-1:], slow, len(prompt) - 1 + i).read()
        truth.append(int(row.argmax()))
    fast = m.caches()
    m.forward(prompt[:-1], fast, 0)
    done, past, steps = 0, len(prompt) - 1, 0
    kv = ctx.kv_list(*fast, m.cap, m.kel, m.vel)
    while done < 30:
        # Up to three true tokens in a row, each among wrong ones; children in a random order.
        n_true = int(rng.integers(0, 4))
        parent, tokens, at = [-1], [truth[done]], 0
        for d in range(3):
            ids = [t for t in rng.integers(0, m.vocab, 3) if t != truth[done + d + 1]]
            if d < n_true:
                ids.insert(int(rng.integers(0, len(ids) + 1)), truth[done + d + 1])
            first = len(parent)
            for t in ids:
                parent.append(at)
                tokens.append(int(t))
            at = first + ids.index(truth[done + d + 1]) if d < n_true else first
        depth, mask = hip.tree_plan(np.array(parent, np.int32))
        n = len(parent)
        logits = m.forward(tokens, fast, past, (ctx.upload(depth), ctx.upload(mask)))
        path, count, nxt = (ctx.empty(4 * k, np.int32) for k in (n, 1, 1))
        ctx.verify_tree(logits, None, ctx.upload(np.array(tokens, np.int32)), ctx.upload(np.array(parent, np.int32)), n, m.vocab,
                        0.0, None, path, count, nxt)
        ctx.kv_gather(kv, past, kv, past, m.layers, m.kv, 64, path, n, count)
        c = int(count.read()[0])
        assert c == n_true + 1
        got = [tokens[j] for j in path.read()[1:c]] + [int(nxt.read()[0])]
        assert got == truth[done + 1:done + 1 + c]
        done, past, steps = done + c, past + c, steps + 1
    assert steps < done
    for i in range(m.layers):
        for a, b, shape in zip(m.at(fast, i), m.at(slow, i), ((m.kv, m.cap, 64), (m.kv, 64, -1))):
            a, b = (x.read(np.float16).reshape(shape).astype(np.float64) for x in (a, b))
            a, b = (x[:, :past] if shape[1] == m.cap else x[..., :past] for x in (a, b))
            # two f32 evaluations of an f16 row: a rounding step apart here and there
            assert np.linalg.norm(a - b) <= 2.0**-11 * np.linalg.norm(b)


def _runtime():
    rt = ctypes.CDLL("libamdhip64.so")
    vp, pvp = ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)
    rt.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    rt.hipStreamEndCapture.argtypes = [vp, pvp]
    rt.hipGraphInstantiate.argtypes = [pvp, vp, vp, vp, ctypes.c_size_t]
    rt.hipGraphLaunch.argtypes = [vp, vp]
    rt.hipGraphExecDestroy.argtypes = [vp]
    rt.hipGraphDestroy.argtypes = [vp]
    return rt


@pytest.mark.parametrize("nodes,past,how", [(9, 80, "lookup"), (40, 1500, "sampled"), (24, 300, "greedy")])
def test_a_captured_step_replays(ctx, hip, nodes, past, how):
    """One layer's step with its verification and gather, captured once and replayed on new inputs,
    with the same calls made directly between the replays: the same bits every time."""
    rng = np.random.default_rng(nodes)
    heads, kv, cap, vocab = 14, 2, past + nodes, 3001
    parent = T.random_tree(rng, nodes)
    depth, mask = hip.tree_plan(parent)
    cos, sin = (ctx.upload(t) for t in hip.rope_tables(64, 1e6, cap))
    par, dep, msk = (ctx.upload(x) for x in (parent, depth, mask))

    def inputs(seed):
        r = np.random.default_rng(seed)
        logits, q, tokens, _, u = _drafts(r, nodes, vocab, how)
        tokens[1:] = np.where(r.random(nodes - 1) < 0.5, logits[parent[1:]].argmax(1), tokens[1:])
        return [r.standard_normal((nodes, h * 64)).astype(np.float32) for h in (heads, kv, kv)] + [logits, q, tokens, u] + \
            [_f16(r, kv, cap, 64), _f16(r, kv, 64, _vstride(cap))]

    bufs = [None if x is None else ctx.upload(x) for x in inputs(0)]
    qr, out = ctx.empty(nodes * heads * 256), ctx.empty(nodes * heads * 256)
    path, count, nxt = (ctx.empty(4 * k, np.int32) for k in (nodes, 1, 1))

    def load(seed):
        for b, x in zip(bufs, inputs(seed)):
            if b is not None:
                x = np.ascontiguousarray(x)
                assert ctx.lib.qh_upload(ctx.handle, b.ptr, x.ctypes.data, x.nbytes) == 0

    def step():
        q, k, v, logits, draft, tokens, u, kc, vc = bufs
        ctx.rope_append_tree(q, k, v, cos, sin, cap, dep, qr, kc, vc, cap, heads, kv, 64, past, nodes)
        ctx.attention_tree(qr, kc, vc, cap, msk, out, nodes, past, heads, kv)
        ctx.verify_tree(logits, draft, tokens, par, nodes, vocab, 0.0 if how == "greedy" else 0.9, u, path, count, nxt)
        c = ctx.kv_list(kc, vc, cap)
        ctx.kv_gather(c, past, c, past, 1, kv, 64, path, nodes, count)

    def results():
        return [b.read(np.uint16).copy() for b in (qr, out, path, count, nxt, bufs[7], bufs[8])]

    rt = _runtime()
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamBeginCapture(ctx.stream, 1) == 0  # thread local
    step()
    assert rt.hipStreamEndCapture(ctx.stream, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    for seed in (1, 2, 3, 1):
        load(seed)
        step()
        want = results()
        load(seed)
        assert rt.hipGraphLaunch(run, ctx.stream) == 0
        for a, b in zip(results(), want):
            np.testing.assert_array_equal(a, b)
    ctx.done()
    rt.hipGraphExecDestroy(run)
    rt.hipGraphDestroy(graph)


# ---------------------------------------------------------- calls side by side --

def _attention_case(ctx, nodes, past, heads, kv, seed):
    rng = np.random.default_rng(seed)
    keys, values = _caches(rng, kv, past + nodes, past + nodes)
    q = rng.standard_normal((nodes, heads * 64)).astype(np.float32)
    _, see = T.plan(T.random_tree(rng, nodes))
    bufs = [ctx.upload(np.ascontiguousarray(x)) for x in (q, keys, values, T.pack(see))] + [ctx.empty(q.nbytes)]

    def call():
        ctx.attention_tree(bufs[0], bufs[1], bufs[2], past + nodes, bufs[3], bufs[4], nodes, past, heads, kv)

    return call, bufs[4]


MIXED = [(5, 100, 14, 2), (64, 12900, 32, 1), (16, 1024, 14, 2), (300, 6000, 20, 4), (3, 9000, 14, 2), (130, 2000, 14, 1)]


def test_scratch_that_grows_between_calls_in_flight(ctx, hip):
    """A context's first calls, small and large, none waited for: the results of calls on their own."""
    own = hip.GpuContext.create(0)
    cases = [_attention_case(own, *shape, seed=i) for i, shape in enumerate(MIXED)]
    own.done()
    for call, _ in cases:
        call()
    first = [out.read() for _, out in cases]
    for (call, out), want in zip(cases, first):
        call()
        np.testing.assert_array_equal(out.read(), want)
    own.close()


def test_two_contexts_on_two_threads(hip):
    """Each thread's context has a stream and scratch of its own."""
    contexts = [hip.GpuContext.create(0) for _ in range(2)]
    cases = [[_attention_case(c, *shape, seed=10 * k + i) for i, shape in enumerate(MIXED)] for k, c in enumerate(contexts)]
    want = []
    for mine in cases:
        want.append([])
        for call, out in mine:
            call()
            want[-1].append(out.read())
    errors = []

    def run(k):
        try:
            for _ in range(5):
                order = np.random.default_rng(k).permutation(len(MIXED))
                for i in order:
                    cases[k][i][0]()
                for i in order:
                    np.testing.assert_array_equal(cases[k][i][1].read(), want[k][i])
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    for c in contexts:
        c.close()


@pytest.mark.parametrize("captured_by,mode", [((0, 1), 1), ((0, 0), 1), ((0, 1), 0)])
def test_two_graphs_side_by_side(hip, captured_by, mode):
    """Two graphs whose calls need scratch, captured by two contexts or by one, replayed at once on two streams, again
    before they have ended, with direct calls between."""
    rt = _runtime()
    contexts = [hip.GpuContext.create(0) for _ in range(2)]
    cases = [[_attention_case(contexts[c], *shape, seed=20 * k + i) for i, shape in enumerate(MIXED)] for k, c in enumerate(captured_by)]
    want, graphs, runs = [], [], []
    for c, mine in zip((contexts[c] for c in captured_by), cases):
        want.append([])
        for call, out in mine:
            call()
            want[-1].append(out.read())
        graph, run = ctypes.c_void_p(), ctypes.c_void_p()
        c.done()
        assert rt.hipStreamBeginCapture(c.stream, mode) == 0  # thread local or global
        for call, _ in mine:
            call()
        assert rt.hipStreamEndCapture(c.stream, ctypes.byref(graph)) == 0
        assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
        graphs.append(graph)
        runs.append(run)
    for turn in range(4):
        for mine in cases:
            for _, out in mine:
                nan = np.full(out.nbytes // 4, np.nan, np.float32)
                assert out.ctx.lib.qh_upload(out.ctx.handle, out.ptr, nan.ctypes.data, nan.nbytes) == 0
        for _ in range(3):
            for c, run in zip(contexts, runs):
                assert rt.hipGraphLaunch(run, c.stream) == 0
        for c in contexts:
            c.done()
        for k, mine in enumerate(cases):
            for (call, out), w in zip(mine, want[k]):
                np.testing.assert_array_equal(out.read(), w)
            if turn % 2:
                mine[turn][0]()
    for c in contexts:
        c.done()
    for graph, run in zip(graphs, runs):
        rt.hipGraphExecDestroy(run)
        rt.hipGraphDestroy(graph)
    for c in contexts:
        c.close()
