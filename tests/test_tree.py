"""Decoding from a tree of drafts, on the CPU: the host helper, the refusals of every entry point
(each is decided before anything is launched), and the law of the 64-bit verification that the
GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import tree_lib as T


@pytest.mark.parametrize("nodes", [1, 2, 63, 64, 65, 200])
def test_tree_plan(hip, nodes):
    parent = T.random_tree(np.random.default_rng(nodes), nodes)
    depth, mask = hip.tree_plan(parent)
    want_depth, see = T.plan(parent)
    np.testing.assert_array_equal(depth, want_depth)
    np.testing.assert_array_equal(mask, T.pack(see))


@pytest.mark.parametrize("parent,what", [([0], "root"), ([-1, 1], "node 1"), ([-1, 0, 5, 0], "node 2"), ([-1, -1], "node 1"),
                                         ([], "nodes")])
def test_tree_plan_refuses_what_is_no_tree(hip, parent, what):
    with pytest.raises(hip.QwenHipError, match=what):
        hip.tree_plan(np.array(parent, np.int32))


class _Fake:
    """A context that no call below gets to use: every refusal comes before it is touched."""

    def __init__(self, hip):
        self.lib, self.block = hip.load_library(), ctypes.create_string_buffer(4096)
        self.handle = ctypes.addressof(self.block)
        raw = ctypes.create_string_buffer(4096 + 64)
        self.raw = raw
        base = (ctypes.addressof(raw) + 63) // 64 * 64
        self.buf = hip.DeviceBuffer(self, base, 4096)
        self.odd = hip.DeviceBuffer(self, base + 4, 4092)
        self.byte = hip.DeviceBuffer(self, base + 2, 4094)


def _refused(hip, call, args, changes, error, what):
    args = {**args, **changes}
    with pytest.raises(error, match=what) as e:
        getattr(hip.GpuContext, call)(_Fake.current, **args)
    assert not isinstance(e.value, hip.RangeError) or error is hip.RangeError


@pytest.fixture
def fake(hip):
    _Fake.current = _Fake(hip)
    return _Fake.current


def test_rope_append_tree_refuses(hip, fake):
    b = fake.buf
    ok = dict(q=b, k=b, v=b, cos=b, sin=b, table_positions=20, depth=b, q_out=b, kc=b, vc=b, capacity=20, heads=4,
              kv_heads=2, head_dim=64, past=10, nodes=5)
    E, R = hip.QwenHipError, hip.RangeError
    for changes, error, what in [({"nodes": 0}, E, "nodes=0"), ({"past": -1}, E, "past=-1"), ({"heads": 0}, E, "heads=0"),
                                 ({"kv_heads": 0}, E, "kv_heads=0"), ({"head_dim": 7}, E, "head_dim=7"),
                                 ({"heads": 1 << 20}, E, "too wide"), ({"past": 16}, R, "cannot add 5"),
                                 ({"past": 2**31 - 1}, R, "cannot add"), ({"table_positions": 14}, R, "rope table"),
                                 ({"capacity": (1 << 30) + 1}, E, "1073741824 positions"),
                                 ({"capacity": 1 << 30, "table_positions": 1 << 30, "past": 0, "nodes": (1 << 22) + 1}, E, "2\\^31 values"),
                                 ({"q": hip.DeviceBuffer(fake, 0, 0)}, E, "needs q"),
                                 ({"vc": hip.DeviceBuffer(fake, 0, 0)}, E, "both caches")]:
        _refused(hip, "rope_append_tree", ok, changes, error, what)


def test_attention_tree_refuses(hip, fake):
    b = fake.buf
    ok = dict(q=b, kc=b, vc=b, capacity=20, mask=b, out=b, nodes=5, past=10, heads=4, kv_heads=2)
    E, R = hip.QwenHipError, hip.RangeError
    for changes, error, what in [({"nodes": 0}, E, "nodes >= 1"), ({"past": -1}, E, "past >= 0"), ({"head_dim": 128}, E, "head_dim 64"),
                                 ({"heads": 5}, E, "group evenly"), ({"kv_heads": 0}, E, "group evenly"),
                                 ({"heads": 1}, E, "group evenly"), ({"past": 16}, R, "exceeds capacity"),
                                 ({"past": 2**31 - 3}, R, "exceeds capacity"),
                                 ({"nodes": 1 << 21, "past": 0, "capacity": 1 << 21}, E, "4194304 rows"),
                                 ({"capacity": (1 << 27) + 1}, E, "134217728 positions"), ({"q": fake.odd}, E, "aligned"),
                                 ({"kc": fake.byte}, E, "aligned"), ({"vc": fake.byte}, E, "aligned"), ({"out": fake.odd}, E, "aligned"),
                                 ({"mask": fake.odd}, E, "aligned"), ({"mask": hip.DeviceBuffer(fake, 0, 0)}, E, "the mask")]:
        _refused(hip, "attention_tree", ok, changes, error, what)


def test_verify_tree_refuses(hip, fake):
    b = fake.buf
    ok = dict(logits=b, draft=None, tokens=b, parent=b, nodes=5, vocab=100, temperature=1.0, uniform=b, path=b, count=b,
              next_token=b)
    E = hip.QwenHipError
    for changes, error, what in [({"nodes": 0}, E, "nodes"), ({"nodes": 1025}, E, "1024 nodes"), ({"vocab": 0}, E, "vocabulary"), ({"vocab": 2**24 + 1}, E, "vocabulary"),
                                 ({"temperature": -0.5}, E, "temperature"), ({"temperature": float("nan")}, E, "temperature"),
                                 ({"temperature": float("inf")}, E, "temperature"), ({"temperature": 1e-40}, E, "temperature"),
                                 ({"uniform": None}, E, "random number"),
                                 ({"count": hip.DeviceBuffer(fake, 0, 0)}, E, "three outputs")]:
        _refused(hip, "verify_tree", ok, changes, error, what)


def test_kv_gather_refuses(hip, fake):
    b = fake.buf

    def kv(key=0, value=1 << 20, capacity=16, ks=0, vs=0):
        return hip.KvList(b.ptr + key, b.ptr + value, ks, vs, capacity)

    far = 1 << 24
    ok = dict(src=kv(), src_base=0, dst=kv(far, far + (1 << 20)), dst_base=0, layers=1, kv_heads=2, head_dim=64, rows=b, n=4)
    E, R = hip.QwenHipError, hip.RangeError
    span = 2 * 16 * 64 * 2
    for changes, error, what in [
            ({"layers": 0}, E, "layers=0"), ({"kv_heads": 0}, E, "kv_heads=0"), ({"head_dim": 12}, E, "head_dim=12"),
            ({"head_dim": 0}, E, "head_dim=0"), ({"n": -1}, E, "n, both bases"), ({"src_base": -1}, E, "bases"),
            ({"dst_base": -1}, E, "bases"), ({"dst_base": 13}, R, "cannot write 4 at 13"),
            ({"dst_base": 2**31 - 1}, R, "cannot write"), ({"src_base": 13, "rows": None}, R, "cannot read 4 at 13"),
            ({"src_base": 17}, R, "cannot read"), ({"src": kv(8)}, E, "aligned"), ({"dst": kv(far, far + 4)}, E, "aligned"),
            ({"src": kv(capacity=2**30 + 1)}, E, "1073741824"), ({"dst": kv(far, far + (1 << 20), 2**31 - 1)}, E, "1073741824"),
            ({"src": kv(capacity=0)}, E, "capacities"), ({"layers": 2}, E, "strides"),
            ({"layers": 2, "src": kv(ks=2052, vs=8192), "dst": kv(far, far + (1 << 20), 16, 2048, 8192)}, E, "strides"),
            ({"src": kv(ks=2**20, vs=2**20), "dst": kv(far, far + (1 << 20), 16, 2040, 8192), "layers": 2}, E, "strides"),
            # overlaps: the same keys under other values, part of the keys, keys over values
            ({"dst": kv(0, far)}, E, "overlap"), ({"dst": kv(span - 16, far)}, E, "overlap"), ({"dst": kv(far, 16)}, E, "overlap"),
            ({"dst": kv(capacity=12)}, E, "overlap"), ({"dst": kv(1 << 20, far)}, E, "overlap")]:
        _refused(hip, "kv_gather", ok, changes, error, what)
    hip.GpuContext.kv_gather(fake, **{**ok, "n": 0})  # nothing to move: accepted, nothing launched


# ------------------------------------------------------------ the law itself --

@pytest.mark.parametrize("how", ["drawn", "given"])
def test_the_walk_keeps_the_targets_distribution(how):
    """The first token that leaves the root is distributed as p, whatever the drafts: over 30000
    trials each of 6 frequencies lies within 5 standard deviations, sqrt(p (1 - p) / trials)."""
    rng = np.random.default_rng(5)
    vocab, trials = 6, 30000
    logits = np.zeros((4, vocab), np.float32)
    logits[0] = [0.3, 1.2, -0.5, 2.0, -np.inf, 0.0]
    logits[1:] = rng.standard_normal((3, vocab))
    draft = np.tile(np.float32([0.1, 0.15, 0.3, 0.2, 0.05, 0.2]), (4, 1))
    parent = np.array([-1, 0, 0, 0], np.int32)
    p = T.weights(logits[0], 0.7)
    p /= p.sum()
    seen = np.zeros(vocab)
    for _ in range(trials):
        drawn = rng.choice(vocab, 3, p=draft[0] / draft[0].sum(dtype=np.float64)) if how == "drawn" else np.array([3, 0, 3])
        tokens = np.concatenate([[0], drawn]).astype(np.int32)
        path, nxt = T.verify(logits, draft if how == "drawn" else None, tokens, parent, 0.7, rng.random(4))
        seen[tokens[path[1]] if len(path) > 1 else nxt] += 1
    np.testing.assert_array_less(np.abs(seen / trials - p), 5 * np.sqrt(p * (1 - p) / trials) + 1e-12)
