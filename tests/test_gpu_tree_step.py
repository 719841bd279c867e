"""Whole verification steps of a drafted tree, as an engine runs them (plan, pre-pass, attention, recurrent layer, commits),
against the same tokens decoded one at a time, and the step captured into a graph."""
import numpy as np
import pytest
import torch

from irontimber_amd import ops
from irontimber_amd.synth import rope_theta_scale
from tests import tree_ref as ref
from tests.gpu_util import announce, dev_f32, host

pytestmark = pytest.mark.gpu
NH, NKV, NV, NK, EPS, K = 16, 2, 32, 16, 1e-6, 4
CD, CTX = (2 * NK + NV) * 128, 400
N_ROT = 64


class Layers:
    """One attention layer's cache and one recurrent layer's states, with their weights."""

    def __init__(self, dev, seed):
        r = np.random.default_rng(seed)
        f = lambda *s: dev_f32(r.standard_normal(s), dev)
        self.kc, self.vc = (torch.zeros(CTX, NKV * 256, device=dev, dtype=torch.float16) for _ in range(2))
        self.state, self.conv, self.conv2 = 0.05 * f(NV, 128, 128), f(K - 1, CD), torch.empty(K - 1, CD, device=dev)
        self.w, self.dt, self.a = 0.5 * f(CD, K), 0.1 * f(NV), -torch.exp(f(NV).clamp(-1, 1))
        self.qn, self.kn = 1 + 0.1 * f(256), 1 + 0.1 * f(256)
        # the model's own rotation as a table
        ts = np.float64(np.float32(rope_theta_scale(1e7, N_ROT)))
        self.freq = dev_f32(ts ** np.arange(N_ROT // 2), dev)


def tokens(r, nt, dev):
    """What the projections of nt tokens hand to the two layers."""
    f = lambda *s: dev_f32(r.standard_normal(s), dev)
    return dict(q=f(nt, NH * 512), k=f(nt, NKV * 256), v=f(nt, NKV * 256), x=f(nt, CD), beta=f(nt, NV), alpha=f(nt, NV))


def decode(m: Layers, t, i, pos):
    """Token i decoded alone at position pos."""
    row = {k: z[i:i + 1].clone() for k, z in t.items()}
    ops.attn_prep_f16(row["q"], row["k"], row["v"], m.kc, m.vc, pos, NH, NKV, m.qn, m.kn, EPS)
    a = ops.attn_f16(row["q"], m.kc, m.vc, pos, NH, NKV)
    g = ops.gdn_decode_fused(row["x"], m.w, m.conv, m.conv2, row["beta"], row["alpha"], m.dt, m.a, m.state, NV, NK, EPS)
    m.conv, m.conv2 = m.conv2, m.conv
    return host(a)[0], host(g)[0]


def tree_step(m: Layers, t, parent, pos0, leaf, trace, scratch):
    """The nodes t of a tree after pos0 committed tokens, and the commit of the path to leaf."""
    nt = len(parent)
    anc, pos = ops.tree_plan(parent, pos0)
    q = t["q"].clone()
    ops.attn_prep_pos_f16(q, t["k"], t["v"], m.kc, m.vc, pos, pos0, NH, NKV, m.freq, q_norm=m.qn, k_norm=m.kn, eps=EPS)
    a = ops.attn_tree_f16(q, m.kc, m.vc, pos0, NH, NKV, anc, scratch=scratch)
    g = ops.gdn_tree(t["x"], m.w, m.conv, t["beta"], t["alpha"], m.dt, m.a, m.state, anc, NV, NK, trace, EPS)
    ops.kv_tree_commit_f16(m.kc, m.vc, pos0, nt, anc, leaf)
    ops.gdn_tree_commit(t["x"], m.conv, m.state, anc, leaf, NV, NK, trace)
    return a, g


def close(got, want, what):
    """f32 arithmetic on both sides, in other orders: 64 steps of the largest value, and for the cache half an f16 step more
    where the two rotations' tables differ by a rounding."""
    assert np.abs(got - want).max() <= 64 * 2.0 ** -20 * np.abs(want).max(), what


@pytest.mark.parametrize("seed", [1, 2])
def test_steps_agree_with_decoding_one_at_a_time(dev, seed):
    r = np.random.default_rng(seed)
    m, one = Layers(dev, seed), Layers(dev, seed)
    pos = 0
    for step, (shape, nt, accept) in enumerate([("chain", 3, 2), ("random", 40, 31), ("star", 7, 4), ("padded", 64, 50),
                                                ("forest", 12, -1), ("random", 64, 63), ("chain", 1, 0), ("padded", 17, 3)]):
        par = ref.parents(shape, nt, seed + step)
        while accept >= 0 and ref.path(par, accept) is None:
            accept -= 1
        announce(f"step {step}: {shape} {nt} at {pos}, accept {accept}")
        t = tokens(r, nt, dev)
        parent = torch.from_numpy(par).to(dev)
        trace = ops.gdn_tree_trace(nt, NV, NK, dev)
        scratch = torch.empty(max(ops.attn_tree_scratch_bytes(pos, nt, NH, NKV), 16), device=dev, dtype=torch.uint8)
        a, g = (host(z) for z in tree_step(m, t, parent, pos, accept, trace, scratch))
        kept = ref.path(par, accept) if accept >= 0 else []
        for i, node in enumerate(kept):
            want_a, want_g = decode(one, t, node, pos + i)
            close(a[node], want_a, f"attention of node {node}")
            close(g[node], want_g, f"recurrence of node {node}")
        pos += len(kept)
        close(host(m.state), host(one.state), "state")
        assert np.array_equal(host(m.conv), host(one.conv))
        # K is rotated by one table and by the other: an f16 step apart at most
        k0, k1 = host(m.kc[:pos]).astype(np.float64), host(one.kc[:pos]).astype(np.float64)
        assert (np.abs(k0 - k1) <= 2.0 ** -10 * np.abs(k1) + 2.0 ** -20).all()
        assert np.array_equal(host(m.vc[:pos]), host(one.vc[:pos]))
        one.kc[:pos] = m.kc[:pos]
    assert pos >= 20


@pytest.mark.parametrize("nt", [5, 33])
def test_captured_step_replays(dev, nt):
    """The step in a graph: parents and inputs change between replays, which give bit for bit what the calls give."""
    r = np.random.default_rng(nt)
    pos0, leaf = 150, 2
    m = Layers(dev, 3)
    m.kc[:pos0].normal_()
    m.vc[:pos0].normal_()
    t, parent = tokens(r, nt, dev), torch.zeros(nt, device=dev, dtype=torch.int32)
    parent.copy_(torch.from_numpy(ref.parents("chain", nt)))
    trace = ops.gdn_tree_trace(nt, NV, NK, dev)
    scratch = torch.empty(ops.attn_tree_scratch_bytes(pos0, nt, NH, NKV), device=dev, dtype=torch.uint8)
    kept = [z.clone() for z in (m.kc, m.vc, m.state, m.conv)]

    def reset():
        for z, old in zip((m.kc, m.vc, m.state, m.conv), kept):
            z.copy_(old)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tree_step(m, t, parent, pos0, leaf, trace, scratch)     # loads the kernels
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = tree_step(m, t, parent, pos0, leaf, trace, scratch)
    for rep, shape in enumerate(["random", "chain", "padded", "star", "random"]):
        fresh = tokens(r, nt, dev)
        for k in t:
            t[k].copy_(fresh[k])
        parent.copy_(torch.from_numpy(ref.parents(shape, nt, rep)))
        reset()
        want = [host(z).copy() for z in tree_step(m, t, parent, pos0, leaf, trace, scratch)]
        want += [host(z).copy() for z in (m.kc, m.vc, m.state, m.conv)]
        reset()
        scratch.fill_(0xFF)
        trace.fill_(0xFF)
        graph.replay()
        got = [host(z) for z in (*out, m.kc, m.vc, m.state, m.conv)]
        for a, b in zip(got, want):
            assert np.array_equal(a, b), f"replay {rep}"


def test_two_steps_at_once(dev):
    """Two sequences' steps on two streams, each with its own scratch and trace: the results of running them in turn."""
    r = np.random.default_rng(9)
    nt, pos0 = 24, 120
    seqs = []
    for seed in (11, 12):
        m = Layers(dev, seed)
        m.kc[:pos0].normal_()
        m.vc[:pos0].normal_()
        seqs.append((m, tokens(r, nt, dev), torch.from_numpy(ref.parents("random", nt, seed)).to(dev),
                     ops.gdn_tree_trace(nt, NV, NK, dev),
                     torch.empty(ops.attn_tree_scratch_bytes(pos0, nt, NH, NKV), device=dev, dtype=torch.uint8)))
    kept = [[z.clone() for z in (m.kc, m.vc, m.state, m.conv)] for m, *_ in seqs]
    run = lambda s: tree_step(s[0], s[1], s[2], pos0, nt - 1, s[3], s[4])
    want = [[host(z).copy() for z in (*run(s), s[0].kc, s[0].vc, s[0].state, s[0].conv)] for s in seqs]
    for s, old in zip(seqs, kept):
        for z, o in zip((s[0].kc, s[0].vc, s[0].state, s[0].conv), old):
            z.copy_(o)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in seqs], []
    for stream, s in zip(streams, seqs):
        with torch.cuda.stream(stream):
            outs.append(run(s))
    torch.cuda.synchronize()
    for s, out, w in zip(seqs, outs, want):
        for a, b in zip([host(z) for z in (*out, s[0].kc, s[0].vc, s[0].state, s[0].conv)], w):
            assert np.array_equal(a, b)
