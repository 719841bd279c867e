"""Attention of a drafted tree's nodes against the f64 statement."""
import numpy as np
import pytest
import torch

from irontimber_amd import _lib, ops
from irontimber_amd.synth import f16_bits, rmsnorm_rows
from tests import tree_ref as ref
from tests.gpu_util import announce, dev_f32, host

pytestmark = pytest.mark.gpu


def inputs(seed, nt, pos0, nh, nkv, kscale=1.0):
    r = np.random.default_rng(seed)
    f = lambda *s: r.standard_normal(s).astype(np.float32)
    rows = pos0 + nt
    k = (rmsnorm_rows(f(rows, nkv, 256)) * kscale).reshape(rows, -1).astype(np.float16)
    return f(nt, nh, 512), k, f(rows, nkv * 256).astype(np.float16)


def run(dev, q, k, v, pos0, nh, nkv, anc, **kw):
    nt = len(q)
    out = torch.full((nt, nh * 256), float("nan"), device=dev)
    ops.attn_tree_f16(dev_f32(q.reshape(nt, -1), dev), torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), pos0, nh,
                      nkv, torch.from_numpy(anc).to(dev), out=out, **kw)
    return host(out).reshape(nt, nh, 256)


def check(dev, seed, nt, pos0, nh, nkv, shape, hidden=None, kscale=1.0, **kw):
    announce(f"attn_tree nt={nt} pos0={pos0} {nh}/{nkv} {shape} {kw}")
    q, k, v = inputs(seed, nt, pos0, nh, nkv, kscale)
    anc = ref.masks(ref.parents(shape, nt, seed))
    want, tol = ref.attn(q, k, v, pos0, nh, nkv, anc, 1 / 16)
    got = run(dev, q, k, v, pos0, nh, nkv, anc, **kw)
    assert (np.abs(got - want) <= tol).all(), float(np.nanmax(np.abs(got - want) - tol))
    assert (got[anc == 0] == 0).all()
    return got


@pytest.mark.parametrize("nh,nkv", [(16, 2), (24, 4), (4, 4), (16, 1), (7, 1)])
@pytest.mark.parametrize("nt,shape", [(1, "chain"), (2, "forest"), (5, "star"), (13, "padded"), (33, "random"), (64, "chain"),
                                      (64, "padded")])
def test_geometries(dev, nh, nkv, nt, shape):
    check(dev, nt, nt, 333, nh, nkv, shape)


@pytest.mark.parametrize("pos0", [0, 1, 2, 31, 63, 64, 65, 127, 128, 129, 1000, 1024, 2049])
@pytest.mark.parametrize("nt", [1, 6, 40])
def test_context_lengths(dev, pos0, nt):
    check(dev, pos0, nt, pos0, 16, 2, "random")


@pytest.mark.parametrize("nt,shape", [(1, "chain"), (4, "star"), (26, "padded"), (64, "random")])
def test_long_context(dev, nt, shape):
    check(dev, 9, nt, 8100, 16, 2, shape)


@pytest.mark.parametrize("nt,pos0,shape", [(1, 20000, "chain"), (2, 9001, "forest"), (3, 300, "star"), (5, 5003, "random"),
                                           (8, 10007, "random"), (26, 1200, "padded"), (40, 2000, "random")])
def test_forms_of_the_context(dev, nt, pos0, shape):
    """8 rows a workgroup with one tile and with several, 16 rows with one (one and two workgroups a CU), two and five, and
    64 rows."""
    check(dev, 21, nt, pos0, 16, 2, shape)


def test_sharp_and_flat_scores(dev):
    """One key takes nearly all the weight (scores up to about 100), and all keys the same (scores of zero)."""
    check(dev, 3, 9, 700, 16, 2, "random", kscale=25.0)
    check(dev, 3, 9, 700, 16, 2, "random", kscale=0.0)


@pytest.mark.parametrize("nt", [3, 20, 64])
def test_scratch_sizes(dev, nt):
    """Any scratch from one record per (node, head) on; the same sums in other splits."""
    pos0, nh = 1500, 16
    full = ops.attn_tree_scratch_bytes(pos0, nt, nh, 2)
    one = nt * nh * 1040
    assert full >= one
    for nbytes in {one, one + 1000, 2 * one, full // 2, full, full + 4096}:
        if nbytes < one:
            continue
        buf = torch.full((nbytes + 64,), 0x7F, device=dev, dtype=torch.uint8)
        check(dev, 5, nt, pos0, nh, 2, "random", scratch=buf[:nbytes])
        assert (host(buf[nbytes:]) == 0x7F).all()
    with pytest.raises(_lib.ItError, match="scratch"):
        check(dev, 5, nt, pos0, nh, 2, "random", scratch=torch.empty(one - 16, device=dev, dtype=torch.uint8))


@pytest.mark.parametrize("pos0", [0, 200])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 65504.0, -65504.0])
def test_hidden_rows_are_not_seen(dev, pos0, bad):
    """Whatever the padding nodes' rows, the rows behind the tree and the other branches' rows hold, a node's output is
    bit for bit the one that it has with zeros there."""
    nt, nh, nkv = 24, 16, 2
    q, k, v = inputs(7, nt, pos0, nh, nkv)
    par = ref.parents("padded", nt, 7)
    anc = ref.masks(par)
    base = run(dev, q, k, v, pos0, nh, nkv, anc)
    dead = [t for t in range(nt) if anc[t] == 0]
    assert len(dead) >= 3
    k2, v2 = k.copy(), v.copy()
    for t in dead:
        k2[pos0 + t], v2[pos0 + t] = bad, bad
    extra = np.full((3, nkv * 256), bad, np.float16)
    assert np.array_equal(run(dev, q, np.concatenate([k2, extra]), np.concatenate([v2, extra]), pos0, nh, nkv, anc), base)
    # one live branch spoilt: the nodes that do not descend from it keep their outputs
    spoilt = next(t for t in range(nt - 1, 0, -1) if anc[t] != 0)
    k2[pos0 + spoilt], v2[pos0 + spoilt] = bad, bad
    got = run(dev, q, k2, v2, pos0, nh, nkv, anc)
    keep = [t for t in range(nt) if not int(anc[t]) >> spoilt & 1]
    assert np.array_equal(got[keep], base[keep])
    if not np.isfinite(bad):
        assert not np.isfinite(got[spoilt]).all()


def test_masks_of_any_bits(dev):
    """Bits at and above nt are ignored; a node may see any of the tree's rows, later ones too."""
    nt, pos0 = 10, 70
    q, k, v = inputs(11, nt, pos0, 16, 2)
    anc = np.array([0x3FF, 1 << 9, 2, 0, -1, 5, 1 << 63 - 1, 8, 0x155, 0x2AA], np.int64)
    seen = anc & 0x3FF
    want, tol = ref.attn(q, k, v, pos0, 16, 2, seen, 1 / 16)
    got = run(dev, q, k, v, pos0, 16, 2, anc)
    assert (np.abs(got - want) <= tol).all() and (got[3] == 0).all() and (got[6] == 0).all()


def test_chain_agrees_with_the_verify_call(dev):
    """A chain is what it_attn_f16 computes for consecutive tokens; both within the bound."""
    nt, pos0 = 4, 777
    q, k, v = inputs(13, nt, pos0, 16, 2)
    anc = ref.masks(ref.parents("chain", nt))
    want, tol = ref.attn(q, k, v, pos0, 16, 2, anc, 1 / 16)
    a = run(dev, q, k, v, pos0, 16, 2, anc)
    b = host(ops.attn_f16(dev_f32(q.reshape(nt, -1), dev), torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), pos0,
                          16, 2)).reshape(nt, 16, 256)
    assert (np.abs(a - want) <= tol).all() and (np.abs(a - b) <= 2 * tol).all()


def test_strides_and_streams(dev):
    """Token strides wider than the rows (what lies between stays), on a stream that is not the default one."""
    nt, pos0, nh, nkv = 7, 130, 16, 2
    q, k, v = inputs(17, nt, pos0, nh, nkv)
    anc = ref.masks(ref.parents("random", nt, 17))
    want, tol = ref.attn(q, k, v, pos0, nh, nkv, anc, 1 / 16)
    qts, ots = nh * 512 + 20, nh * 256 + 12
    wide = np.zeros((nt, qts), np.float32)
    wide[:, :nh * 512] = q.reshape(nt, -1)
    args = [dev_f32(wide, dev), torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), torch.from_numpy(anc).to(dev)]
    out = torch.full((nt, ots), 7.0, device=dev)
    scr = torch.empty(ops.attn_tree_scratch_bytes(pos0, nt, nh, nkv), device=dev, dtype=torch.uint8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    _lib.call("it_attn_tree_f16", args[0].data_ptr(), qts, args[1].data_ptr(), args[2].data_ptr(), 512, pos0, 256, nh, nkv,
              nt, nt, args[3].data_ptr(), 1 / 16, out.data_ptr(), ots, scr.data_ptr(), scr.numel(), s.cuda_stream)
    got = host(out)
    assert (got[:, nh * 256:] == 7.0).all()
    assert (np.abs(got[:, :nh * 256].reshape(nt, nh, 256) - want) <= tol).all()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_levels_of_a_draft(dev, kv):
    """The nodes of each depth asked for on their own, with the rows drafted so far, get what all nodes at once get."""
    nt, pos0, nh, nkv = 20, 90, 16, 2
    q, k, v = inputs(19, nt, pos0, nh, nkv)
    if kv == "f32":
        k, v = k.astype(np.float32), v.astype(np.float32)
    par = ref.parents("random", nt, 19)
    par[12:] = np.sort(par[12:])
    anc = ref.masks(par)
    call = ops.attn_tree_f16 if kv == "f16" else ops.attn_tree_f32kv
    qd, kd, vd = dev_f32(q.reshape(nt, -1), dev), torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
    ad = torch.from_numpy(anc).to(dev)
    want, tol = ref.attn(q, k, v, pos0, nh, nkv, anc, 1 / 16)
    for a, b in ((0, 1), (1, 5), (5, 12), (12, 20)):
        # what lies behind the rows drafted so far is not there yet
        got = host(call(qd[a:b], kd[:pos0 + b], vd[:pos0 + b], pos0, nh, nkv, ad[a:b], rows=b)).reshape(b - a, nh, 256)
        assert (np.abs(got - want[a:b]) <= tol[a:b]).all()


@pytest.mark.parametrize("nh,nkv", [(16, 2), (24, 4), (4, 4), (16, 1)])
@pytest.mark.parametrize("nt,pos0,shape", [(1, 0, "chain"), (1, 1, "chain"), (2, 63, "forest"), (3, 64, "star"), (5, 65, "star"),
                                           (13, 500, "padded"), (33, 333, "random"), (64, 1000, "padded"),
                                           (64, 2049, "chain")])
def test_f32_cache(dev, nh, nkv, nt, pos0, shape):
    announce(f"attn_tree_f32kv nt={nt} pos0={pos0} {nh}/{nkv} {shape}")
    r = np.random.default_rng(nt + pos0)
    f = lambda *s: r.standard_normal(s).astype(np.float32)
    q, k, v = f(nt, nh, 512), f(pos0 + nt, nkv * 256), f(pos0 + nt, nkv * 256)
    anc = ref.masks(ref.parents(shape, nt, nt))
    want, tol = ref.attn(q, k, v, pos0, nh, nkv, anc, 1 / 16)
    k[pos0:][anc == 0], v[pos0:][anc == 0] = np.nan, np.nan     # a padding node's rows are not looked at
    args = (dev_f32(q.reshape(nt, -1), dev), dev_f32(k, dev), dev_f32(v, dev), pos0, nh, nkv, torch.from_numpy(anc).to(dev))
    full = ops.attn_tree_f32kv_scratch_bytes(pos0, nt, nh, nkv)
    for nbytes in {full, nt * nh * 1040 if pos0 else 0}:
        out = torch.full((nt, nh * 256), float("nan"), device=dev)
        ops.attn_tree_f32kv(*args, out=out, scratch=torch.empty(nbytes, device=dev, dtype=torch.uint8))
        got = host(out).reshape(nt, nh, 256)
        assert (np.abs(got - want) <= tol).all() and (got[anc == 0] == 0).all()


def test_offsets_past_32_bits(dev):
    """The longest context (2^22 rows, 4 GiB a cache): offsets beyond 2^31 elements in the context and the tree."""
    nt, nh, nkv = 6, 16, 2
    pos0 = (1 << 22) - nt
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    k, v = (torch.randn(pos0 + nt, nkv * 256, device=dev, generator=g, dtype=torch.float16) for _ in range(2))
    q = torch.randn(nt, nh, 512, device=dev, generator=g)
    # the last rows matter most: the keys after 2^31 elements point along the queries of the first head of their group
    q[:, :, :256] *= 0.02
    k[-40:] = q[0, [0, 8], :256].reshape(-1).half() * 400
    anc = ref.masks(ref.parents("random", nt, 2))
    got = ops.attn_tree_f16(q.view(nt, -1), k, v, pos0, nh, nkv, torch.from_numpy(anc).to(dev)).view(nt, nh, 256)
    for kh in range(nkv):
        heads = slice(8 * kh, 8 * kh + 8)
        for t in (0, nt - 1):
            own = torch.tensor([pos0 + j for j in range(nt) if int(anc[t]) >> j & 1], device=dev)
            qt = q[t, heads, :256].double()
            col = slice(256 * kh, 256 * kh + 256)
            parts = [k[a:min(a + (1 << 19), pos0), col] for a in range(0, pos0, 1 << 19)] + [k[own, col]]
            vals = [v[a:min(a + (1 << 19), pos0), col] for a in range(0, pos0, 1 << 19)] + [v[own, col]]
            s = [qt @ x.double().T.contiguous() / 16 for x in parts]
            m = torch.stack([x.amax(-1) for x in s]).amax(0)[:, None]
            l = sum(torch.exp(x - m).sum(-1) for x in s)[:, None]
            o = sum(torch.exp(x - m) @ y.double() for x, y in zip(s, vals)) / l
            want = o * torch.sigmoid(q[t, heads, 256:].double())
            # as in the statement: scores (up to 6 here), weights in two f16 a key, sums
            tol = (2 * (20 * 6 + 4) + 32) * 2.0 ** -24 * 6 + (1 << 22) * 2.0 ** -25 / l * 6
            assert ((got[t, heads].double() - want).abs() <= tol).all()
