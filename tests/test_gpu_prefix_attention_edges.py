"""k3xb_prefix_attention where its fast forms end.

Tolerances as in test_gpu_prefix_attention.py: 2 u of sum p |v| for
probabilities and outputs rounded to the type (u = 2^-8 bf16, 2^-11 f16), 1e-5
of it for float scores and sums.
"""
import ctypes as C
import math

import pytest

from gpu_util import torch_cuda
from test_gpu_prefix_attention import _case, _chain, _check, _run

pytestmark = pytest.mark.gpu

F16 = 2.0 ** -11


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


def _flat_tail(torch, ctx, S, N, prefix, own, sink):
    """One position (of the prefix, or of the own rows where there is none)
    25.5 powers of two above all others, which hold the value 1: what they add up
    to is the output."""
    q = torch.zeros(S, N, 1, 64, dtype=torch.float16, device="cuda")
    q[..., 0] = 16.0
    k, v = (torch.zeros(prefix or own, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    k[sink, 0, 0] = 25.5 * math.log(2.0) * 8.0 / 16.0   # the scale is 1 / 8
    v[:] = 1.0
    v[sink] = 0.0
    score = float(k[sink, 0, 0]) * 16.0 / 8.0
    small = torch.zeros(1, N, 1, 64, dtype=torch.float16, device="cuda")
    suffix = [(torch.cat([t, small[0]]) if not prefix else small[0])[None].expand(S, -1, -1, -1) for t in (k, v)]
    out = torch.empty(S, N, 1, 64, dtype=torch.float16, device="cuda")
    lens = torch.full((S,), 0 if prefix else own, dtype=torch.int32, device="cuda")
    ctx.prefix_attention(q, k if prefix else None, v if prefix else None, suffix[0], suffix[1], lens, [-1] * N, out)
    ctx.sync()
    n = (prefix or own) - 1
    want = n / (math.exp(score) + n + 1)   # the node itself holds the value 0
    err = float((out.double() - want).abs().max())
    assert err <= (2.0 * F16 + 1e-5) * want, (err, want)


@pytest.mark.parametrize("sink", [0, 199999, 399999])
def test_f16_flat_tail_of_a_long_prefix(torch, ctx, sink):
    """Rows for every SM to see the whole prefix."""
    _flat_tail(torch, ctx, 600, 64, 400000, 0, sink)


@pytest.mark.parametrize("sink", [0, 15000])
def test_f16_flat_tail_of_own_rows(torch, ctx, sink):
    """Sequences enough for one task to see all of one's rows."""
    _flat_tail(torch, ctx, 6000, 1, 0, 20000, sink)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_long_flat_sums(torch, ctx, kind):
    """As many equal positions as one task may sum: rows for every SM to see
    the whole prefix. Every value is 0.7 of 11 (8) bits: a float sum of them is not exact."""
    dtype = getattr(torch, kind)
    S, N, rows = 600, 64, 700000
    q, own = (torch.zeros(S, N, 1, 64, dtype=dtype, device="cuda") for _ in range(2))
    k, v = (torch.full((rows, 1, 64), x, dtype=dtype, device="cuda") for x in (0.0, 0.7))
    out = torch.empty(S, N, 1, 64, dtype=dtype, device="cuda")
    lse = torch.empty(S, N, 1, device="cuda")
    ctx.prefix_attention(q, k, v, own, own + v[0], torch.zeros(S, dtype=torch.int32, device="cuda"), [-1] * N, out, lse=lse)
    ctx.sync()
    want = float(v[0, 0, 0])
    err = float((out.double() - want).abs().max()) / want
    assert err <= 2.0 * (F16 if kind == "float16" else 2.0 ** -8) + 1e-5, err
    assert float((lse.double() - math.log(rows + 1)).abs().max()) <= 1e-5


@pytest.mark.parametrize("heads,kv_heads,main,extra,value", [(8, 8, 128, 64, 128), (16, 2, 64, 0, 64), (16, 1, 128, 64, 128)])
@pytest.mark.parametrize("N", [1, 4, 9])
@pytest.mark.parametrize("prefix", [400, 1024, 1025, 3333])
def test_one_sequence(torch, ctx, heads, kv_heads, main, extra, value, N, prefix):
    """A short prefix goes with the own rows, a long one on its own."""
    c = _case(torch, 1, N, heads, kv_heads, main, extra, value, prefix, [37], "bfloat16", 950 + prefix + N)
    _check(torch, ctx, c, _chain(N))


@pytest.mark.parametrize("S,heads,kv_heads,lens", [(3, 4, 2, [0, 700, 5000]), (5, 8, 8, [1100, -1, 15, 2600, 511]), (300, 8, 4, [3, 600, 1500, 0, 77])])
@pytest.mark.parametrize("prefix", [0, 333])
@pytest.mark.parametrize("spare", [0, 9000])
def test_roomy_caches(torch, ctx, S, heads, kv_heads, lens, prefix, spare):
    """Sequences of unlike lengths in caches with room for far longer ones: some
    become several tasks, some one, some none."""
    lens = [lens[i % len(lens)] for i in range(S)]
    spare = spare if S < 100 else min(spare, 900)
    c = _case(torch, S, 2, heads, kv_heads, 64, 64, 64, prefix, lens, "bfloat16", 970 + S + prefix, spare=spare)
    _check(torch, ctx, c, _chain(2))


@pytest.mark.parametrize("kind,el", [("bfloat16", 2), ("float16", 2), ("float32", 4)])
def test_arrays_off_their_alignment_are_refused(torch, ctx, kind, el):
    """Refused on the host: no kernel sees such a pointer."""
    import k3xb
    c = _case(torch, 2, 2, 4, 2, 64, 64, 64, 30, [3, 4], kind, 940)
    lens = torch.tensor(c["lens"], dtype=torch.int32).cuda()
    out = torch.empty(2, 2, 4, 64, dtype=c["q"].dtype, device="cuda")
    lse = torch.empty(2, 2, 4, device="cuda")
    parent = (C.c_int32 * 2)(-1, 0)
    io = k3xb.PrefixAttentionIO(sequences=2, nodes=2, heads=4, kv_heads=2, main_dim=64, extra_dim=64, value_dim=64,
                                type={"float32": 0, "bfloat16": 1, "float16": 2}[kind], scale=0.1,
                                parent=C.addressof(parent), q=c["q"].data_ptr(), suffix_len=lens.data_ptr(), out=out.data_ptr(),
                                lse=lse.data_ptr())
    for src, rows in ((io.prefix, "prefix"), (io.suffix, "suffix")):
        src.k, src.v, src.extra = (c[rows + n].data_ptr() for n in ("_k", "_v", "_extra"))
        src.rows = c[rows + "_k"].shape[-3]
    call = ctx.lib.k3xb_prefix_attention
    assert call(ctx.h, C.byref(io)) == 0
    ctx.sync()
    clean = out.clone()
    out.fill_(7.0)
    torch.cuda.synchronize()
    for obj, field, step in [(io, "q", el), (io, "out", el), (io, "lse", 4), (io, "suffix_len", 4)] + [
            (src, n, el) for src in (io.prefix, io.suffix) for n in ("k", "v", "extra")]:
        at = getattr(obj, field)
        for shift in range(1, step):
            setattr(obj, field, at + shift)
            assert call(ctx.h, C.byref(io)) == k3xb.INVALID_EXTENT, (field, shift)
        setattr(obj, field, at)
    io.type = 3
    assert call(ctx.h, C.byref(io)) == k3xb.INVALID_EXTENT
    ctx.sync()
    assert bool((out == 7.0).all())
    io.type = {"float32": 0, "bfloat16": 1, "float16": 2}[kind]
    assert call(ctx.h, C.byref(io)) == 0
    ctx.sync()
    assert torch.equal(out, clean)


@pytest.mark.parametrize("S", [2, 3])
def test_prefix_past_32_bits(torch, ctx, S):
    """The tensor maps step over more than 2^31 key elements; the last rows decide."""
    rows, heads = 530000, 32
    q = torch.zeros(S, 1, heads, 128, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 16.0
    k = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    k[-1, :, 0] = 30.0
    v[-1] = torch.arange(heads, device="cuda").to(torch.bfloat16)[:, None]
    own = torch.zeros(S, 2, heads, 128, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(S, 1, heads, 128, dtype=torch.bfloat16, device="cuda")
    ctx.prefix_attention(q, k, v, own, own, torch.zeros(S, dtype=torch.int32).cuda(), [-1], out)
    ctx.sync()
    weight = 1.0 / (1.0 + rows * math.exp(-480.0 / math.sqrt(128)))
    want = weight * torch.arange(heads, dtype=torch.float64, device="cuda")[:, None].expand(heads, 128)
    assert bool(((out[:, 0].double() - want).abs() <= 2.0 ** -7 * want).all())


@pytest.mark.parametrize("kind,heads,rows", [("bfloat16", 32, 190000), ("bfloat16", 33, 190000), ("float32", 3, 1900000)])
def test_own_rows_past_32_bits(torch, ctx, kind, heads, rows):
    """The last sequence's last rows lie past 2^31 elements, and decide."""
    S, dtype = 3, getattr(torch, kind)
    q = torch.zeros(S, 1, heads, 128, dtype=dtype, device="cuda")
    q[..., 0] = 16.0
    k, v = (torch.zeros(S, rows, heads, 128, dtype=dtype, device="cuda") for _ in range(2))
    k[:, -2, :, 0] = 30.0
    v[:, -2] = torch.arange(1, heads + 1, device="cuda").to(dtype)[:, None]
    v[:, -1] = 5.0   # the node's own row
    out = torch.empty(S, 1, heads, 128, dtype=dtype, device="cuda")
    lens = torch.tensor([3, 1000, rows - 1], dtype=torch.int32)
    ctx.prefix_attention(q, None, None, k, v, lens.cuda(), [-1], out)
    ctx.sync()
    far = math.exp(-480.0 / math.sqrt(128))
    total = 1.0 + (rows - 1) * far
    want = (torch.arange(1, heads + 1, dtype=torch.float64, device="cuda")[:, None].expand(heads, 128) + 5.0 * far) / total
    assert bool(((out[2, 0].double() - want).abs() <= 2.0 ** -7 * want).all())
    assert not out[:2].any()


@pytest.mark.parametrize("S,lens", [(3, [1500, 20, 900]), (1, [40])])
def test_in_a_graph(torch, ctx, S, lens):
    """All launch forms of a call, replayed on other inputs and lengths."""
    c = _case(torch, S, 2, 4, 2, 128, 64, 128, 700, lens, "bfloat16", 990 + S, spare=600)
    other = _case(torch, S, 2, 4, 2, 128, 64, 128, 700, lens[::-1], "bfloat16", 991 + S, spare=600)
    want, want_lse = _run(torch, ctx, other, _chain(2))
    device = torch.tensor(c["lens"], dtype=torch.int32).cuda()
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)

    def call():
        ctx.prefix_attention(c["q"], c["prefix_k"], c["prefix_v"], c["suffix_k"], c["suffix_v"], device, _chain(2), out,
                             prefix_extra=c["prefix_extra"], suffix_extra=c["suffix_extra"], lse=lse)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.use_stream(side)
        try:
            call()
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                call()
        finally:
            ctx.use_stream()
    for n in ("q", "prefix_k", "prefix_v", "prefix_extra", "suffix_k", "suffix_v", "suffix_extra"):
        c[n].copy_(other[n])
    device.copy_(torch.tensor(other["lens"], dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
