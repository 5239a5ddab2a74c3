"""Attention over a shared prefix, own rows and draft ancestors
(k3xb_prefix_attention) against its formula in 64 bits.

Tolerances, with u the unit roundoff of the type (2^-8 bf16, 2^-11 f16): the
probabilities may be rounded to the type and the output is, so a value is off
by at most 2 u of sum p |v|, and float scores and sums add 1e-5 of it. A
score is a float sum of at most 256 products, off by 256 * 2^-24 = 1.5e-5 of
the sum of its terms' sizes; lse inherits that.
"""
import math

import numpy as np
import pytest

from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


@pytest.fixture(scope="module")
def torch():
    return torch_cuda()


@pytest.fixture(scope="module")
def ctx(torch):
    import k3xb
    c = k3xb.Context(0)
    c.use_stream()
    yield c
    c.close()


def _chain(n):
    return [i - 1 for i in range(n)]


def _tree(n):
    return [-1 if i == 0 else (i - 1) // 2 for i in range(n)]


def _forest(n):
    return [-1 if i % 3 == 0 else i - 1 for i in range(n)]


def _case(torch, S, N, heads, kv_heads, main, extra, value, prefix, lens, kind, seed, spare=2, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    dtype = getattr(torch, kind)
    cap = max(0, *lens) + N + spare

    def rnd(*shape, s=1.0):
        return (s * torch.randn(*shape, generator=g)).to(dtype).cuda()

    c = dict(q=rnd(S, N, heads, main + extra, s=2.0 * spread), prefix_k=rnd(prefix, kv_heads, main),
             prefix_v=rnd(prefix, kv_heads, value), suffix_k=rnd(S, cap, kv_heads, main),
             suffix_v=rnd(S, cap, kv_heads, value), prefix_extra=rnd(prefix, extra) if extra else None,
             suffix_extra=rnd(S, cap, extra) if extra else None, lens=list(lens))
    return c


def _formula(torch, c, parent, scale=None):
    """(out, lse, sum p |v|, sum of |score terms|) in 64 bits."""
    q = c["q"].double()
    S, N, heads, width = q.shape
    main, g = c["suffix_k"].shape[-1], heads // c["suffix_k"].shape[2]
    scale = 1.0 / math.sqrt(width) if scale is None else scale
    value = c["suffix_v"].shape[-1]
    out = torch.zeros(S, N, heads, value, dtype=torch.float64, device="cuda")
    size, lse = out.clone(), torch.full((S, N, heads), -math.inf, dtype=torch.float64, device="cuda")
    terms = torch.zeros_like(lse)
    for s, n_own in enumerate(c["lens"]):
        if n_own < 0:
            continue
        for n in range(N):
            own, j = list(range(n_own)), n
            while j >= 0:
                own.append(n_own + j)
                j = parent[j]
            k = torch.cat([c["prefix_k"], c["suffix_k"][s, own]]).double().repeat_interleave(g, 1)
            v = torch.cat([c["prefix_v"], c["suffix_v"][s, own]]).double().repeat_interleave(g, 1)
            if c["prefix_extra"] is not None:
                e = torch.cat([c["prefix_extra"], c["suffix_extra"][s, own]]).double()
                k = torch.cat([k, e[:, None, :].expand(-1, heads, -1)], dim=-1)
            x = scale * torch.einsum("hd,phd->hp", q[s, n], k)
            terms[s, n] = abs(scale) * torch.einsum("hd,phd->hp", q[s, n].abs(), k.abs()).amax(-1)
            lse[s, n] = torch.logsumexp(x, -1)
            p = torch.exp(x - lse[s, n][:, None])
            out[s, n] = torch.einsum("hp,phv->hv", p, v)
            size[s, n] = torch.einsum("hp,phv->hv", p, v.abs())
    return out, lse, size, terms


def _run(torch, ctx, c, parent, scale=None):
    S, N, heads, _ = c["q"].shape
    out = torch.full((S, N, heads, c["suffix_v"].shape[-1]), 7.0, dtype=c["q"].dtype, device="cuda")
    lse = torch.full((S, N, heads), 7.0, device="cuda")
    ctx.prefix_attention(c["q"], c["prefix_k"], c["prefix_v"], c["suffix_k"], c["suffix_v"],
                         torch.tensor(c["lens"], dtype=torch.int32).cuda(), parent, out, prefix_extra=c["prefix_extra"],
                         suffix_extra=c["suffix_extra"], lse=lse, scale=scale)
    ctx.sync()
    return out, lse


def _check(torch, ctx, c, parent, scale=None):
    out, lse = _run(torch, ctx, c, parent, scale)
    want, want_lse, size, terms = _formula(torch, c, parent, scale)
    u = UNIT[str(c["q"].dtype).split(".")[1]]
    score = 1.5e-5 * terms + 1e-6 * (1.0 + want_lse.abs().nan_to_num(0.0, posinf=0.0))
    live = torch.tensor(c["lens"], device="cuda") >= 0
    err = (out.double() - want).abs()
    bound = (2.0 * u + 1e-5 + 2.0 * score[..., None]) * size
    assert torch.isfinite(out).all() and bool((err <= bound).all()), \
        f"worst {float((err - bound).max()):.3e} past its bound, of {float(size.max()):.3e}"
    dl = (lse.double() - want_lse).abs()[live]
    assert bool((dl <= score[live]).all()), f"lse off by {float(dl.max()):.3e}"
    assert not out[~live].any() and bool((lse[~live] == -math.inf).all())
    return out, lse


SHAPES = [  # heads, kv_heads, main, extra, value
    (3, 3, 128, 64, 128), (4, 2, 128, 0, 128), (8, 1, 64, 0, 64), (2, 2, 64, 64, 64), (6, 2, 128, 64, 64), (2, 1, 64, 64, 128),
    (2, 2, 8, 4, 8), (3, 1, 40, 0, 24), (2, 2, 192, 64, 256),   # the general form
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
def test_shapes(torch, ctx, shape, kind):
    heads, kv_heads, main, extra, value = shape
    c = _case(torch, 3, 5, heads, kv_heads, main, extra, value, 150, [37, 0, 130], kind, 3 + main + extra + heads)
    _check(torch, ctx, c, _tree(5))


@pytest.mark.parametrize("prefix", [0, 1, 2, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_prefix_lengths(torch, ctx, prefix):
    c = _case(torch, 2, 3, 2, 2, 128, 64, 128, prefix, [5, 0], "bfloat16", 100 + prefix)
    _check(torch, ctx, c, _chain(3))


@pytest.mark.parametrize("lens", [[0], [1], [127, 128, 129], [-1, 0, 300], [-1, -1], [64, 63, 65, -3, 256, 2]], ids=str)
@pytest.mark.parametrize("prefix", [0, 77])
def test_own_lengths(torch, ctx, lens, prefix):
    c = _case(torch, len(lens), 2, 4, 2, 128, 0, 128, prefix, lens, "bfloat16", 200 + prefix + len(lens))
    _check(torch, ctx, c, _chain(2))


@pytest.mark.parametrize("nodes,topology", [(1, _chain), (2, _forest), (9, _chain), (17, _tree), (32, _tree), (33, _forest),
                                            (64, _chain), (64, _tree)])
def test_topologies(torch, ctx, nodes, topology):
    c = _case(torch, 2, nodes, 2, 1, 64, 64, 64, 70, [3, 20], "float16", 300 + nodes)
    _check(torch, ctx, c, topology(nodes))


@pytest.mark.parametrize("S,N,heads,kv_heads", [(1, 1, 1, 1), (1, 1, 64, 1), (43, 3, 2, 2), (86, 3, 2, 1), (5, 7, 16, 2), (130, 1, 2, 2),
                                               (300, 1, 1, 1), (29, 9, 2, 2)])
def test_row_counts(torch, ctx, S, N, heads, kv_heads):
    """Rows of a kv head, S * N * group, below, at and past whole tiles."""
    c = _case(torch, S, N, heads, kv_heads, 128, 64, 128, 300, [(7 * s) % 11 for s in range(S)], "bfloat16", 400 + S)
    _check(torch, ctx, c, _chain(N))


def test_long_prefix(torch, ctx):
    c = _case(torch, 2, 2, 2, 2, 128, 64, 128, 20011, [700, 9], "bfloat16", 500)
    _check(torch, ctx, c, _chain(2))


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
def test_peaked_and_flat_scores(torch, ctx, kind):
    """Scores from a few hundred apart (one position takes all) to equal, the
    largest ones late and early, so that the running maximum moves a lot."""
    for spread, seed in ((60.0, 1), (0.0, 2)):
        c = _case(torch, 2, 4, 2, 2, 128, 0, 128, 700, [300, 1], kind, 600 + seed, spread=spread)
        ramp = torch.linspace(0.0, 1.0, 700, device="cuda")[:, None, None]
        for flip in (False, True):
            c["prefix_k"] = (c["prefix_k"].float() * (ramp.flip(0) if flip else ramp)).to(c["q"].dtype)
            _check(torch, ctx, c, _chain(4))


def test_negative_and_zero_scale(torch, ctx):
    c = _case(torch, 2, 2, 2, 2, 64, 0, 64, 140, [30, 0], "bfloat16", 610)
    _check(torch, ctx, c, _chain(2), scale=-0.2)
    _check(torch, ctx, c, _chain(2), scale=0.0)


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), 1e38])
@pytest.mark.parametrize("shape", [(2, 2, 128, 64, 128), (2, 2, 8, 4, 8)], ids=str)
def test_rows_that_are_not_visible_do_not_matter(torch, ctx, junk, shape):
    """Rows past a sequence's own, drafts off a node's path and idle
    sequences hold anything."""
    heads, kv_heads, main, extra, value = shape
    parent = [-1, 0, 0, 1]
    c = _case(torch, 4, 4, heads, kv_heads, main, extra, value, 100, [70, 0, -1, 128], "bfloat16", 700, spare=140)
    clean, clean_lse = _check(torch, ctx, c, parent)
    for s, n in enumerate(c["lens"]):
        first = 0 if n < 0 else n + 4
        for t in (c["suffix_k"], c["suffix_v"], c["suffix_extra"]):
            t[s, first:] = junk
    for t in (c["suffix_k"], c["suffix_v"]):
        t[0, 72] = junk      # node 2 of sequence 0: on no path but its own
    out, lse = _run(torch, ctx, c, parent)
    keep = [0, 1, 3]
    assert torch.equal(out[1:], clean[1:]) and torch.equal(lse[1:], clean_lse[1:])
    assert torch.equal(out[0, keep], clean[0, keep]) and torch.equal(lse[0, keep], clean_lse[0, keep])


def test_nothing_visible_but_itself(torch, ctx):
    """No prefix, no rows: a root's output is its own value."""
    c = _case(torch, 3, 1, 2, 2, 128, 64, 128, 0, [0, 0, 0], "bfloat16", 720)
    out, _ = _check(torch, ctx, c, [-1])
    assert torch.equal(out[:, 0], c["suffix_v"][:, 0])


@pytest.mark.parametrize("order", ["heads first", "interleaved", "odd rows"])
def test_cache_orders(torch, ctx, order):
    """Head-major caches, key and value interleaved per head (as kv_b
    projects them), and rows that no 16-byte load can start at."""
    c = _case(torch, 3, 3, 4, 2, 128, 64, 128, 200, [40, 7, 129], "bfloat16", 800)
    want, want_lse = _run(torch, ctx, c, _chain(3))
    d = dict(c)
    for src in ("prefix", "suffix"):
        k, v = c[src + "_k"], c[src + "_v"]
        if order == "heads first":
            d[src + "_k"], d[src + "_v"] = (t.transpose(-3, -2).contiguous().transpose(-3, -2) for t in (k, v))
        elif order == "interleaved":
            kv = torch.cat([k, v], dim=-1)
            d[src + "_k"], d[src + "_v"] = kv[..., :128], kv[..., 128:]
        else:
            wide = torch.zeros(*k.shape[:-1], 131, dtype=k.dtype, device="cuda")
            wide[..., 1:129] = k
            d[src + "_k"] = wide[..., 1:129]
    if order == "odd rows":
        _check(torch, ctx, d, _chain(3))
    else:
        out, lse = _run(torch, ctx, d, _chain(3))
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("S", [1, 5])
def test_broadcast_caches(torch, ctx, S):
    """One cache for all sequences, one head's rows for all heads, one row for
    all positions: zero strides are taken as they are."""
    N, heads = 2, 4
    c = _case(torch, S, N, heads, heads, 128, 64, 128, 70, [9] * S, "bfloat16", 950)
    for src in ("prefix", "suffix"):
        lead = [] if src == "prefix" else [slice(None)]
        for which in ("cache", "heads", "rows"):
            d = dict(c)
            for n in ("_k", "_v", "_extra"):
                t = c[src + n]
                if which == "cache":
                    if src == "prefix":
                        continue
                    d[src + n] = t[:1].expand_as(t)
                elif which == "heads":
                    if n != "_extra":
                        d[src + n] = t[..., :1, :].expand_as(t)
                else:
                    d[src + n] = t[tuple(lead + [slice(0, 1)])].expand_as(t)
            _check(torch, ctx, d, _chain(N))


def test_offsets_past_32_bits(torch, ctx):
    """A prefix of more than 2^31 key elements whose last rows decide."""
    rows, heads = 530000, 32
    q = torch.zeros(1, 1, heads, 128, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 16.0
    k = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    k[-1, :, 0] = 30.0
    v[-1] = torch.arange(heads, device="cuda").to(torch.bfloat16)[:, None]
    sk = torch.zeros(1, 2, heads, 128, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(1, 1, heads, 128, dtype=torch.bfloat16, device="cuda")
    ctx.prefix_attention(q, k, v, sk, sk, torch.zeros(1, dtype=torch.int32).cuda(), [-1], out)
    ctx.sync()
    weight = 1.0 / (1.0 + rows * math.exp(-480.0 / math.sqrt(128)))
    want = weight * torch.arange(heads, dtype=torch.float64, device="cuda")[:, None].expand(heads, 128)
    assert bool(((out[0, 0].double() - want).abs() <= 2.0 ** -7 * want).all())


def test_streams_and_determinism(torch, ctx):
    c = _case(torch, 9, 5, 4, 2, 128, 64, 128, 900, [30] * 9, "bfloat16", 900)
    a = _run(torch, ctx, c, _chain(5))
    b = _run(torch, ctx, c, _chain(5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ctx.use_stream(side)
    try:
        with torch.cuda.stream(side):
            d = _run(torch, ctx, c, _chain(5))
    finally:
        ctx.use_stream()
    for x in (b, d):
        assert torch.equal(a[0], x[0]) and torch.equal(a[1], x[1])


def test_without_lse(torch, ctx):
    c = _case(torch, 2, 2, 2, 2, 64, 0, 64, 50, [3, 4], "bfloat16", 910)
    want, _ = _run(torch, ctx, c, _chain(2))
    out = torch.empty_like(want)
    ctx.prefix_attention(c["q"], c["prefix_k"], c["prefix_v"], c["suffix_k"], c["suffix_v"],
                         torch.tensor(c["lens"], dtype=torch.int32).cuda(), _chain(2), out)
    ctx.sync()
    assert torch.equal(out, want)


def test_length_past_the_capacity_is_reported(torch, ctx):
    import k3xb
    c = _case(torch, 2, 2, 2, 2, 128, 0, 128, 40, [6, 6], "bfloat16", 920, spare=0)
    want, _ = _run(torch, ctx, c, _chain(2))
    c["lens"] = [6, 7]
    out = torch.full_like(want, 7.0)
    ctx.prefix_attention(c["q"], c["prefix_k"], c["prefix_v"], c["suffix_k"], c["suffix_v"],
                         torch.tensor(c["lens"], dtype=torch.int32).cuda(), _chain(2), out)
    with pytest.raises(k3xb.K3xbError) as e:
        ctx.sync()
    assert e.value.status == k3xb.INVALID_EXTENT
    assert torch.equal(out[0], want[0]) and not out[1].any()
    ctx.sync()


def test_mla_restatement(torch, ctx, rs):
    """The reference's layer at its default widths (the golden fixture's
    weights): the f32 form over its own keys, between the projections of the
    pinned restatement and its gate and output projection (done here)."""
    import os
    z = np.load(os.path.join(os.path.dirname(__file__), "golden", "mla.npz"))
    from test_mla_oracle import _weights
    w = _weights(z)
    x = z["x"]
    T, split = len(x), len(x) - 2
    want, st = rs.mla_prefill(w, x)
    heads, main, extra, value = (int(w[n]) for n in ("heads", "q_main", "q_extra", "value_dim"))
    keys = np.asarray(st["keys"]).reshape(-1, heads, main)[:T]
    values = np.asarray(st["values"]).reshape(-1, heads, value)[:T]
    shared = np.asarray(st["shared"]).reshape(-1, extra)[:T]

    def norm(v, g):
        v = v.astype(np.float64)
        return v / np.sqrt((v * v).mean(-1, keepdims=True) + w["eps"]) * g

    q = norm(x.astype(np.float64) @ w["q_a_proj"].T.astype(np.float64), w["q_a_norm"]) @ w["q_b_proj"].T.astype(np.float64)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()   # noqa: E731
    out = torch.empty(1, 2, heads, value, device="cuda")
    ctx.prefix_attention(dev(q[split:]).view(1, 2, heads, main + extra), dev(keys[:split]), dev(values[:split]),
                         dev(keys[None, split:]), dev(values[None, split:]), torch.zeros(1, dtype=torch.int32).cuda(), [-1, 0],
                         out, prefix_extra=dev(shared[:split]), suffix_extra=dev(shared[None, split:]))
    ctx.sync()
    gate = 1.0 / (1.0 + np.exp(-(x[split:].astype(np.float64) @ w["g_proj"].T.astype(np.float64))))
    got = (out[0].cpu().numpy().astype(np.float64).reshape(2, -1) * gate) @ w["o_proj"].T.astype(np.float64)
    # float scores and a float softmax on both sides
    np.testing.assert_allclose(got, np.asarray(want)[split:], rtol=0, atol=2e-5 * np.abs(want).max())


def test_refusals(torch, ctx):
    import k3xb
    c = _case(torch, 2, 2, 4, 2, 64, 64, 64, 30, [3, 4], "bfloat16", 930)
    lens = torch.tensor(c["lens"], dtype=torch.int32).cuda()
    out = torch.empty(2, 2, 4, 64, dtype=torch.bfloat16, device="cuda")

    def call(parent=(-1, 0), lens=lens, out=out, lse=None, scale=None, **kw):
        d = {**c, **kw}
        ctx.prefix_attention(d["q"], d["prefix_k"], d["prefix_v"], d["suffix_k"], d["suffix_v"], lens, list(parent), out,
                             prefix_extra=d["prefix_extra"], suffix_extra=d["suffix_extra"], lse=lse, scale=scale)

    call()
    wrong = [dict(parent=(0, -1)), dict(parent=(-1, 1)), dict(parent=(-2, 0)), dict(parent=(-1,)), dict(lens=lens.long()), dict(lens=lens[:1]),
             dict(lens=lens.cpu()), dict(out=out.float()), dict(out=out[:1]), dict(lse=torch.empty(2, 2, 3, device="cuda")),
             dict(q=c["q"].double()), dict(q=c["q"][:, :, :3].contiguous(), out=out[:, :, :3].contiguous()),
             dict(prefix_k=c["prefix_k"].half()), dict(prefix_extra=None), dict(suffix_extra=None),
             dict(suffix_k=c["suffix_k"][:, :1], suffix_v=c["suffix_v"][:, :1], suffix_extra=c["suffix_extra"][:, :1]),
             dict(prefix_v=c["prefix_v"][:-1]), dict(scale=float("nan")), dict(scale=float("inf")),
             dict(prefix_k=c["prefix_k"].repeat_interleave(2, -1)[..., ::2])]
    for i, kw in enumerate(wrong):
        with pytest.raises(k3xb.K3xbError) as e:
            call(**kw)
        assert e.value.status == k3xb.INVALID_EXTENT, (i, kw)
    wide = _case(torch, 1, 65, 1, 1, 64, 0, 64, 0, [0], "bfloat16", 931)
    with pytest.raises(k3xb.K3xbError):
        _run(torch, ctx, wide, _chain(65))
    wide = _case(torch, 1, 1, 1, 1, 200, 64, 64, 0, [0], "bfloat16", 932)
    with pytest.raises(k3xb.K3xbError):
        _run(torch, ctx, wide, [-1])
    assert ctx.lib.k3xb_prefix_attention(ctx.h, None) == k3xb.INVALID_EXTENT
    ctx.sync()
