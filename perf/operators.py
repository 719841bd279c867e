"""The verification of a drafted token tree, as cases that can be timed and checked.

The user is the engine of cases.py with several draft candidates a step. Its model mixes Gated-DeltaNet layers
and softmax attention layers, in the two head geometries of the tests and the benchmark: 16 query / 2 KV heads
with 32 value / 16 key heads in the recurrence, and 24 / 4 with 48 / 16. A tree is up to 64 nodes in topological
order; anc[t] is the 64-bit mask of node t and its ancestors among them (0: a padding node), pos[t] its position.

ops of a case:
  prep     per-head norm and position rotation of q and k at given positions, and the append of k and v to the
           cache (`kv`: f16 or f32), for a tree or for a prompt (`tree` empty: consecutive positions). `layout`:
           rotated pairs in halves or interleaved; `scaled`: frequencies for contexts `factor` times as long
  attn     attention of the tree's nodes over `pos0` cached rows and their own ancestors
  gdn      a recurrent layer over the tree's nodes, and, where `accept` says so, the states after one of them
  keep     the cache rows of the accepted path moved together
"""
from __future__ import annotations

import math
import random

import torch

own = False

HD, S, KC = 256, 128, 4            # head_dim, recurrent state size, conv taps
EPS = 1e-6
BASE, N_ROT = 1e7, 64


def _prep(name, nt, p0, nh=16, nkv=2, hd=HD, n_rot=N_ROT, layout="half", scaled="none", factor=1.0, kv="f16", tree="",
          row0=0):
    return dict(name=name, op="prep", nt=nt, p0=p0, nh=nh, nkv=nkv, hd=hd, n_rot=n_rot, layout=layout, scaled=scaled,
                factor=factor, kv=kv, tree=tree, dead=0, row0=row0)


def _attn(name, nt, pos0, nh=16, nkv=2, tree="beam", dead=0):
    return dict(name=name, op="attn", nt=nt, pos0=pos0, nh=nh, nkv=nkv, tree=tree, dead=dead)


def _gdn(name, nt, nv=32, nk=16, tree="beam", dead=0, accept="deepest"):
    return dict(name=name, op="gdn", nt=nt, nv=nv, nk=nk, tree=tree, dead=dead, accept=accept)


def _keep(name, nt, pos0, nkv=2, tree="beam"):
    return dict(name=name, op="keep", nt=nt, pos0=pos0, nkv=nkv, tree=tree, dead=0)


def listed():
    return [
        # one token of a chat whose cache rows are not its positions any more: latency
        _prep("prep_1_far", 1, 120_000, tree="chain", row0=4095),
        # a tree's nodes in the larger geometry, interleaved pairs, over the MTP head's f32 cache
        _prep("prep_tree_37_f32_24h", 37, 5003, nh=24, nkv=4, layout="interleaved", scaled="ntk", factor=4.0, kv="f32",
              tree="beam", row0=64),
        # the longest prompt in one call, on a context stretched sixteen times: the bytes of q, k and v
        _prep("prep_prompt_8192", 8192, 90_001, scaled="yarn", factor=16.0),
        # a first draft with two alternatives a step, at a short context
        _attn("attn_5_600", 5, 600),
        # a mid-sized tree in a captured batch with padding nodes, the larger geometry, an odd context
        _attn("attn_26_2997_24h", 26, 2997, nh=24, nkv=4, tree="random", dead=5),
        # the largest tree after a long conversation
        _attn("attn_64_8128", 64, 8128),
        # a tree over a context of document size: the cache's bytes and the matrix work
        _attn("attn_64_131072", 64, 131_072, tree="random"),
        # the accepted token and two alternatives through a recurrent layer; the better one is kept
        _gdn("gdn_3", 3, tree="star"),
        # a mid-sized tree with padding in the larger geometry, the deepest branch kept
        _gdn("gdn_26_48v", 26, nv=48, tree="random", dead=5),
        # the largest tree, nothing beyond the first node accepted
        _gdn("gdn_64", 64, accept="first"),
        # a short path of a small tree kept in the cache
        _keep("keep_7", 7, 4001),
        # a whole chain with a rejected first alternative: every row moves
        _keep("keep_64_24h", 64, 8000, nkv=4, tree="shifted"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prep", "prep", "attn", "attn", "attn", "gdn", "gdn", "keep"])
    nh, nkv, nv, nk = rng.choice([(16, 2, 32, 16), (24, 4, 48, 16)])
    tree = rng.choice(["beam", "random", "star", "chain"])
    nt = _log(rng, 1, 64)
    dead = rng.randint(0, nt // 4)
    if op == "attn":
        return {k: v for k, v in _attn("", nt, _log(rng, 1, 65_536), nh, nkv, tree, dead).items() if k != "name"}
    if op == "gdn":
        return {k: v for k, v in _gdn("", nt, nv, nk, tree, dead, rng.choice(["first", "deepest", "none"])).items()
                if k != "name"}
    if op == "keep":
        return {k: v for k, v in _keep("", max(2, nt), _log(rng, 1, 8000), nkv, tree).items() if k != "name"}
    hd = rng.choice([128, 256])
    c = _prep("", nt, _log(rng, 1, 1_000_000), nh, nkv, hd, rng.choice([64, 128, hd]), rng.choice(["half", "interleaved"]),
              rng.choice(["none", "linear", "ntk", "yarn"]), rng.choice([2.0, 8.0, 32.0]), rng.choice(["f16", "f16", "f32"]),
              tree, rng.randint(0, 500))
    if rng.random() < 0.5:
        c.update(tree="", nt=_log(rng, 16, 8192 if nh == 16 else 4096))
    c.pop("name")
    return c


# ---- inputs: those of a model's projections, normal values; K unit-RMS per head as a norm leaves it

def _parents(case, seed):
    """The tree of a case: the parent of each node among the nodes before it, -1 after the last committed token,
    -2 for a padding node."""
    rng, nt, kind = random.Random(seed * 1009 + 17), case["nt"] - case["dead"], case["tree"]
    if kind == "chain":
        p = [t - 1 for t in range(nt)]
    elif kind == "star":            # one accepted token, the alternatives after it
        p = [-1] + [0] * (nt - 1)
    elif kind == "shifted":         # two alternatives at once, all drafts after the second
        p = [-1, -1] + [t - 1 for t in range(2, nt)]
    elif kind == "beam":            # levels of up to eight nodes
        p, last = [-1], [0]
        while len(p) < nt:
            level = range(len(p), min(nt, len(p) + min(8, 2 * len(last))))
            p += sorted(rng.choice(last) for _ in level)
            last = list(level)
    else:                           # any shape: each node after one of the last twelve
        p = [-1] + [rng.randrange(max(-1, t - 12), t) for t in range(1, nt)]
    return p[:nt] + [-2] * case["dead"]


def _tree(case, seed):
    """anc [nt], and for host use: the parents, the live nodes of each depth, the path to the accepted node."""
    parents = _parents(case, seed)
    masks, depth = [], []
    for t, p in enumerate(parents):
        masks.append(0 if p == -2 else (1 << t) | (masks[p] if p >= 0 else 0))
        depth.append(-1 if p == -2 else depth[p] + 1 if p >= 0 else 0)
    levels = [[t for t, d in enumerate(depth) if d == k] for k in range(max(depth) + 1)]
    leaf = {"first": 0, "none": -1}.get(case.get("accept", "deepest"), levels[-1][0])
    path = [] if leaf < 0 else [t for t in range(leaf + 1) if masks[leaf] >> t & 1]
    signed = [m - (1 << 64) if m >> 63 else m for m in masks]
    to = dict(dtype=torch.int64, device="cuda")
    return dict(anc=torch.tensor(signed, **to), depth=torch.tensor(depth, **to), parents=parents, leaf=leaf,
                levels=[torch.tensor(x, **to) for x in levels],
                above=[torch.tensor([parents[t] + 1 for t in x], **to) for x in levels],
                path=torch.tensor(path, **to))


def _freqs(case):
    """The angle of one position for each rotated pair, and the factor of the rotated values."""
    n, kind, factor = case["n_rot"], case["scaled"], case["factor"]
    i = torch.arange(n // 2, dtype=torch.float64)
    base = BASE * factor ** (n / (n - 2)) if kind == "ntk" else BASE
    f, m = base ** (-2 * i / n), 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "yarn":            # pairs of few turns over 8192 positions stretched, those of many kept
        at = lambda turns: n * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(BASE))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), n - 1)
        stretch = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f, m = f / factor * stretch + f * (1 - stretch), 0.1 * math.log(factor) + 1
    return f.float().cuda(), m


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    nt, st = c["nt"], dict(case=c)
    if c["op"] == "gdn":
        nv, nk = c["nv"], c["nk"]
        cd = (2 * nk + nv) * S
        st.update(state=0.02 * n(nv, S, S), w=0.5 * n(cd, KC), conv=n(KC - 1, cd), x=n(nt, cd), beta=n(nt, nv),
                  alpha=n(nt, nv), a=-torch.exp(2 * torch.rand(nv, device="cuda", generator=g) - 1),
                  dt=0.1 * n(nv), out=torch.empty(nt, nv * S, device="cuda"), **_tree(c, seed))
        return st
    if c["op"] == "prep":
        hd, kvd = c["hd"], c["nkv"] * c["hd"]
        kind = torch.float16 if c["kv"] == "f16" else torch.float32
        st.update(q=2 * n(nt, c["nh"] * 2 * hd), k=2 * n(nt, kvd), v=n(nt, kvd), qn=1 + 0.1 * n(hd), kn=1 + 0.1 * n(hd),
                  kc=n(c["row0"] + nt, kvd).to(kind), vc=n(c["row0"] + nt, kvd).to(kind))
        depth = _tree(c, seed)["depth"] if c["tree"] else torch.arange(nt, device="cuda")
        st["pos"] = (c["p0"] + depth).to(torch.int32)
        st["freq"], st["mscale"] = _freqs(c)
        return st
    rows, nkv = c["pos0"] + nt, c["nkv"]
    k = n(rows, nkv, HD)
    st.update(kc=(k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS)).view(rows, -1).half(),
              vc=n(rows, nkv * HD).half(), **_tree(c, seed))
    if c["op"] == "attn":
        st.update(q=n(nt, c["nh"] * 2 * HD), out=torch.empty(nt, c["nh"] * HD, device="cuda"))
    return st


def run(st):
    c = st["case"]
    if c["op"] == "prep":
        (_prep_own if own else _prep_plain)(c, st)
        return dict(q=st["q"], k=st["kc"], v=st["vc"])
    if c["op"] == "attn":
        return _attn_own(c, st) if own else _attn_plain(c, st)
    if c["op"] == "gdn":
        out = _gdn_own(c, st) if own else _gdn_plain(c, st)
        return dict(out=out, state=st["state"], conv=st["conv"])
    (_keep_own if own else _keep_plain)(c, st)
    return dict(k=st["kc"], v=st["vc"])


# ---- the calls of a user's program

def _prep_own(c, st):
    from irontimber_amd import ops
    call = ops.attn_prep_pos_f16 if c["kv"] == "f16" else ops.attn_prep_pos_f32kv
    call(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["pos"], c["row0"], c["nh"], c["nkv"], st["freq"],
         mscale=st["mscale"], layout=c["layout"], q_norm=st["qn"], k_norm=st["kn"], eps=EPS)


def _attn_own(c, st):
    from irontimber_amd import ops
    if "scratch" not in st:         # an engine's arena
        need = ops.attn_tree_scratch_bytes(c["pos0"], c["nt"], c["nh"], c["nkv"])
        st["scratch"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return ops.attn_tree_f16(st["q"], st["kc"], st["vc"], c["pos0"], c["nh"], c["nkv"], st["anc"], out=st["out"],
                             scratch=st["scratch"])


def _gdn_own(c, st):
    from irontimber_amd import ops
    if "trace" not in st:           # held from the layer's call to the commit
        st["trace"] = ops.gdn_tree_trace(c["nt"], c["nv"], c["nk"], st["x"].device)
    out = ops.gdn_tree(st["x"], st["w"], st["conv"], st["beta"], st["alpha"], st["dt"], st["a"], st["state"], st["anc"],
                       c["nv"], c["nk"], st["trace"], EPS, out=st["out"])
    if st["leaf"] >= 0:
        ops.gdn_tree_commit(st["x"], st["conv"], st["state"], st["anc"], st["leaf"], c["nv"], c["nk"], st["trace"])
    return out


def _keep_own(c, st):
    from irontimber_amd import ops
    ops.kv_tree_commit_f16(st["kc"], st["vc"], c["pos0"], c["nt"], st["anc"], st["leaf"])


# ---- the same in elementary operations

def _rotate(x, cos, sin, n_rot, layout):
    """Rotates the first n_rot dims of x [nt, heads, hd] by the angles of each token and pair."""
    r = x[..., :n_rot]
    a, b = (r[..., :n_rot // 2], r[..., n_rot // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    cos, sin = cos[:, None, :], sin[:, None, :]
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.cat(y, -1) if layout == "half" else torch.stack(y, -1).flatten(-2)
    return torch.cat([y, x[..., n_rot:]], -1)


def _prep_plain(c, st):
    nt, hd, row0 = c["nt"], c["hd"], c["row0"]
    angle = st["pos"].double()[:, None] * st["freq"].double()[None, :]
    cos, sin = (angle.cos() * st["mscale"]).float(), (angle.sin() * st["mscale"]).float()
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    q = st["q"].view(nt, c["nh"], 2 * hd)
    q[..., :hd] = _rotate(norm(q[..., :hd], st["qn"]), cos, sin, c["n_rot"], c["layout"])
    k = _rotate(norm(st["k"].view(nt, c["nkv"], hd), st["kn"]), cos, sin, c["n_rot"], c["layout"])
    st["kc"][row0:] = k.reshape(nt, -1).to(st["kc"].dtype)
    st["vc"][row0:] = st["v"].to(st["vc"].dtype)


def _attn_plain(c, st):
    nt, pos0, nh, nkv = c["nt"], c["pos0"], c["nh"], c["nkv"]
    q = st["q"].view(nt, nkv, nh // nkv, 2 * HD)
    heads = lambda x: x.float().view(-1, nkv, HD).transpose(0, 1).contiguous()
    rows = q[..., :HD].permute(1, 0, 2, 3).reshape(nkv, -1, HD)
    s = torch.matmul(rows, heads(st["kc"]).transpose(1, 2).contiguous()) / math.sqrt(HD)
    s = s.view(nkv, nt, nh // nkv, -1)
    sees = (st["anc"][:, None] >> torch.arange(nt, device="cuda")) & 1 == 1
    live = (st["anc"] != 0)[None, :, None, None]
    s[..., pos0:] = s[..., pos0:].masked_fill(~sees[None, :, None, :], -math.inf)
    s = torch.where(live, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(live, m, 0.0))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nkv, -1, p.shape[-1]), heads(st["vc"])).view(nkv, nt, -1, HD) / torch.where(live, l, 1.0)
    return (o.permute(1, 0, 2, 3) * torch.sigmoid(q[..., HD:])).reshape(nt, -1)


def _gdn_plain(c, st):
    nt, nv, nk = c["nt"], c["nv"], c["nk"]
    node = torch.arange(nt, device="cuda")
    bits = (st["anc"][:, None] >> node) & 1 == 1
    # row t, tap j: the input j tokens before node t on its own path, from the conv state beyond the path's start
    depth = bits.sum(1) - 1
    order = torch.where(bits, node[None, :] + KC - 1, -1).sort(1, descending=True)[0]
    order = torch.cat([order, torch.full((nt, KC), -1, device="cuda")], 1)[:, :KC]
    back = torch.arange(KC, device="cuda")[None, :]
    rows = torch.where(back <= depth[:, None], order, (KC + depth[:, None] - 1 - back).clamp(0, KC - 2))
    seen = torch.cat([st["conv"], st["x"]])
    y = (seen[rows] * st["w"].t().flip(0)[None]).sum(1)
    y = (y * torch.sigmoid(y)).view(nt, -1, S)
    qk = y[:, :2 * nk]
    qk = qk / qk.square().sum(-1, keepdim=True).sqrt().clamp_min(EPS)
    head = torch.arange(nv, device="cuda") % nk
    q, k, v = qk[:, :nk][:, head], qk[:, nk:][:, head], y[:, 2 * nk:]
    beta = torch.sigmoid(st["beta"])
    z = st["alpha"] + st["dt"]
    decay = torch.exp(torch.where(z > 20, z, torch.log1p(torch.exp(z))) * st["a"])
    states = torch.empty(nt + 1, nv, S, S, device="cuda")
    states[0] = st["state"]
    out = torch.zeros(nt, nv, S, device="cuda")
    for at, above in zip(st["levels"], st["above"]):      # the recurrence, all nodes of a depth at once
        s = states[above] * decay[at][:, :, None, None]
        delta = (v[at] - (s * k[at][..., None]).sum(2)) * beta[at][..., None]
        s = s + k[at][..., None] * delta[:, :, None, :]
        out[at] = (s * q[at][..., None]).sum(2) / math.sqrt(S)
        states[at + 1] = s
    if st["leaf"] >= 0:
        st["state"].copy_(states[st["leaf"] + 1])
        st["conv"].copy_(torch.cat([st["conv"], st["x"][st["path"]]])[-(KC - 1):])
    return out.view(nt, -1)


def _keep_plain(c, st):
    at = c["pos0"] + st["path"]
    for cache in (st["kc"], st["vc"]):
        cache[c["pos0"]:c["pos0"] + len(at)] = cache[at]


def work(case):
    """Each input read once and each output written once; the products over the keys that a node sees."""
    c, nt = case, case["nt"]
    live = nt - c["dead"]
    if c["op"] == "gdn":
        nv, cd, f = c["nv"], (2 * c["nk"] + c["nv"]) * S, 4
        once = nv * S * S + (KC - 1) * cd + cd * KC
        if c["accept"] != "none":
            once += nv * S * S + (KC - 1) * cd
        return {"bytes": f * (nt * (cd + 2 * nv) + nt * nv * S + once) + 8 * nt, "flops": live * (nv * 7 * S * S + 2 * KC * cd)}
    if c["op"] == "prep":
        kvd, size = c["nkv"] * c["hd"], 2 if c["kv"] == "f16" else 4
        return {"bytes": nt * (2 * c["nh"] * c["hd"] * 4 + 2 * kvd * (4 + size) + 4),
                "flops": nt * (c["nh"] + c["nkv"]) * (4 * c["hd"] + 3 * c["n_rot"])}
    if c["op"] == "keep":
        return {"bytes": 2 * 2 * 2 * nt * c["nkv"] * HD, "flops": 0}
    # q and gate in, out; the cache in; scores and sums over the context and about half of the tree
    b = nt * c["nh"] * HD * 4 * 3 + 2 * (c["pos0"] + nt) * c["nkv"] * HD * 2 + 8 * nt
    return {"bytes": b, "flops": 4 * HD * c["nh"] * live * (c["pos0"] + live / 2)}


# ---- the same in 64 bits

def _ancestors(parents, t):
    path = []
    while t >= 0:
        path.append(t)
        t = parents[t]
    return path[::-1]


def exact(case, seed):
    c, st = dict(case), prepare(case, seed)
    nt = c["nt"]
    if c["op"] == "keep":
        path = _ancestors(st["parents"], st["leaf"])
        moved = lambda x: torch.cat([x[:c["pos0"]], *(x[c["pos0"] + t][None] for t in path), x[c["pos0"] + len(path):]])
        return dict(k=moved(st["kc"].double()), v=moved(st["vc"].double()))
    if c["op"] == "prep":
        hd, half = c["hd"], c["n_rot"] // 2
        turn = torch.polar(torch.full((nt, half), st["mscale"], dtype=torch.float64, device="cuda"),
                           torch.outer(st["pos"].double(), st["freq"].double()))

        def rows(x, heads, w):
            x = x.double().reshape(nt, heads, hd)
            x = x * w.double() / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
            i = torch.arange(half, device="cuda")
            first, second = (i, i + half) if c["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
            x[..., first], x[..., second] = z.real, z.imag
            return x

        q = st["q"].double().view(nt, c["nh"], 2 * hd)
        q = torch.cat([rows(q[..., :hd], c["nh"], st["qn"]), q[..., hd:]], -1).view(nt, -1)
        k = torch.cat([st["kc"][:c["row0"]].double(), rows(st["k"], c["nkv"], st["kn"]).view(nt, -1)])
        return dict(q=q, k=k, v=torch.cat([st["vc"][:c["row0"]].double(), st["v"].double()]))
    parents = st["parents"]
    if c["op"] == "attn":
        nh, nkv, pos0 = c["nh"], c["nkv"], c["pos0"]
        out = torch.zeros(nt, nh, HD, dtype=torch.float64, device="cuda")
        q = st["q"].double().view(nt, nh, 2 * HD)
        for j in range(nkv):
            k, v = (x.view(-1, nkv, HD)[:, j].double() for x in (st["kc"], st["vc"]))
            mine = slice(j * (nh // nkv), (j + 1) * (nh // nkv))
            for t in range(nt):
                if parents[t] == -2:
                    continue
                at = torch.tensor([pos0 + a for a in _ancestors(parents, t)], device="cuda")
                s = torch.cat([k[:pos0], k[at]]) @ q[t, mine, :HD].T.contiguous() / math.sqrt(HD)
                w = torch.softmax(s, 0).T.contiguous()
                out[t, mine] = w[:, :pos0] @ v[:pos0] + w[:, pos0:] @ v[at]
        return (out * torch.sigmoid(q[..., HD:])).view(nt, -1)
    nv, nk = c["nv"], c["nk"]
    w, conv, x = st["w"].double(), st["conv"].double(), st["x"].double()
    out = torch.zeros(nt, nv, S, dtype=torch.float64, device="cuda")
    kept, windows = {-1: st["state"].double()}, {-1: conv}
    head = [h % nk for h in range(nv)]
    for t in range(nt):
        if parents[t] == -2:
            continue
        window = torch.cat([windows[parents[t]], x[t:t + 1]])
        windows[t] = window[1:]
        y = torch.nn.functional.silu((window * w.T).sum(0)).view(-1, S)
        q, k, v = y[:nk][head], y[nk:2 * nk][head], y[2 * nk:]
        q, k = (z / z.norm(dim=-1, keepdim=True).clamp_min(EPS) for z in (q, k))
        decay = torch.exp(torch.nn.functional.softplus(st["alpha"][t].double() + st["dt"].double()) * st["a"].double())
        s = kept[parents[t]] * decay[:, None, None]
        new = (v - torch.matmul(k[:, None], s)[:, 0]) * torch.sigmoid(st["beta"][t].double())[:, None]
        kept[t] = s + k[:, :, None] * new[:, None, :]
        out[t] = torch.matmul(q[:, None], kept[t])[:, 0] / math.sqrt(S)
    return dict(out=out.view(nt, -1), state=kept[st["leaf"]], conv=windows[st["leaf"]])
