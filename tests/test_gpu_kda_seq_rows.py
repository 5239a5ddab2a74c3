"""k3xb_kda_prefill value by value: every token's row of outputs and every row
of the state against the rule in 64 bits, with inputs whose tokens differ by
many orders of magnitude, infinities and NaN.

Tolerances. Let R be a value row's content without cancellation: a token takes
it to max(a) R + |beta| (|v| + |S| |a k|) |k| (2-norms over the key channels; R
starts at the row's norm). A sum of 128 float products is off by at most 128 *
2^-24 = 7.6e-6 of its terms' size, so a row of the state is off by 1e-5 R (as a
2-norm) and an output by 1e-5 R |q|: R up to that token only, since no output
depends on a later one. A bf16 output is rounded once more, by 2^-8 of itself.
Products below the smallest normal float may vanish: 256 * 2^-126 at most.
"""
import math

import numpy as np
import pytest

from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

TOL = 1e-5
FLOOR = 256.0 * 2.0 ** -126
NAMES = ["q", "k", "v", "log_decay", "beta"]


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


def _inputs(torch, T, h, d, seed, gate="mixed"):
    """q, k, v, log_decay [T][h][d] and beta [T][h], float."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(T, h, d, generator=g) for _ in range(3))
    q, k = q / q.norm(dim=-1, keepdim=True), k / k.norm(dim=-1, keepdim=True)
    ld = {"none": torch.zeros(T, h, d),
          "mixed": -5.0 * torch.sigmoid(2.0 * torch.randn(1, h, d, generator=g) - 3.0 + torch.randn(T, h, d, generator=g)),
          # every channel loses 2 to 5 (natural) of itself with each token
          "fast": -2.0 - 3.0 * torch.rand(T, h, d, generator=g),
          "strong": -200.0 * torch.rand(T, h, d, generator=g)}[gate]
    return [t.cuda() for t in (q, k, v, ld, torch.rand(T, h, generator=g))]


def _state(torch, S, h, d, seed=5):
    return torch.randn(S, h, d, d, generator=torch.Generator().manual_seed(seed)).cuda()


def _rule(torch, x, state):
    """(out, state, content at each token [T][h][d], content at the end) of one sequence in 64 bits."""
    q, k, v, ld, beta = (t.double() for t in x)
    s = state.double()
    out, size = torch.zeros_like(v), torch.zeros_like(v)
    R = s.norm(dim=-1)
    for t in range(q.shape[0]):
        a = ld[t].exp()
        s = s * a[:, None, :]
        pred = (s * k[t][:, None, :]).sum(-1)
        R = R * a.amax(-1, keepdim=True) + beta[t][:, None].abs() * (
            v[t].abs() + s.norm(dim=-1) * k[t].norm(dim=-1, keepdim=True)) * k[t].norm(dim=-1, keepdim=True)
        s = s + ((v[t] - pred) * beta[t][:, None])[:, :, None] * k[t][:, None, :]
        out[t] = (s * q[t][:, None, :]).sum(-1)
        size[t] = R * q[t].norm(dim=-1, keepdim=True)
    return out, s, size, R


def _prefill(torch, ctx, x, lengths, state, dtype=None):
    T, h, d = x[0].shape
    flat = [t.reshape(T, h * d) for t in x[:4]]
    flat[:3] = [t.to(dtype or torch.float32) for t in flat[:3]]
    off = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32).cuda()
    out = torch.full((T, h * d), 7.0, dtype=flat[0].dtype, device="cuda")
    new = torch.full((len(lengths), h, d, d), 7.0, device="cuda")
    ctx.kda_prefill(*flat, x[4], off, out, state=state, state_out=new)
    ctx.sync()
    return out.view(T, h, d), new


def _check(torch, got, want, size, what, lead):
    """Where the rule gives a finite value, `got` is within its bound; where it does not, neither is `got`."""
    fin = torch.isfinite(want)
    assert bool((torch.isfinite(got) == fin).all()), \
        f"{what}: finite at other places, first {(torch.isfinite(got) != fin).nonzero()[0].tolist()}"
    bound = TOL * size + FLOOR
    if got.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * want.abs()
    err = (got.double() - want).abs()
    if lead == "state":
        fin = fin.all(-1)
        err = err.norm(dim=-1)
    bad = fin & (~(err <= bound))
    if bool(bad.any()):
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what} at {at}: error {float(err[at]):.3e} > {float(bound[at]):.3e}; {int(bad.sum())} places")


def _run(torch, ctx, x, lengths, state, dtype=None):
    if dtype is not None:   # the values that the call gets
        x = [t.to(dtype).float() if i < 3 else t for i, t in enumerate(x)]
    out, new = _prefill(torch, ctx, x, lengths, state, dtype)
    first = 0
    for s, n in enumerate(lengths):
        w = slice(first, first + n)
        o, st, size, R = _rule(torch, [t[w] for t in x], state[s])
        _check(torch, out[w], o, size, f"out of sequence {s}", "out")
        _check(torch, new[s], st, R, f"state of sequence {s}", "state")
        first += n
    return out, new


@pytest.mark.parametrize("gate", ["mixed", "none", "fast", "strong"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_rows(torch, ctx, gate, d, kind):
    x = _inputs(torch, 118, 2, d, 1 + d, gate)
    _run(torch, ctx, x, [47, 71], _state(torch, 2, 2, d), getattr(torch, kind))


@pytest.mark.parametrize("scale", [1e-35, 1e-32, 1e-30, 1e-27, 1e-20, 1e25])
@pytest.mark.parametrize("where", ["all", "one value channel", "state only", "state below large values"])
def test_small_and_large_values(torch, ctx, scale, where):
    """The rule is linear in v and the state, and a value channel does not see the others."""
    x = _inputs(torch, 60, 2, 128, 11)
    state = _state(torch, 1, 2, 128)
    rows = slice(37, 38) if where == "one value channel" else slice(None)
    if not where.startswith("state"):
        x[2][..., rows] *= scale
    elif where != "state only":
        x[2] *= 1e10
    state[..., rows, :] *= scale
    _run(torch, ctx, x, [60], state)


@pytest.mark.parametrize("gate", ["mixed", "none", "fast"])
@pytest.mark.parametrize("which,low,high", [("q", -10, 10), ("k", -8, 0), ("v", -10, 10), ("beta", -10, 0), ("all", -6, 0)])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_tokens_of_unlike_size(torch, ctx, gate, which, low, high, kind):
    x = _inputs(torch, 75, 2, 128, 17, gate)
    g = torch.Generator().manual_seed(len(which) + high)
    for i, n in enumerate(NAMES):
        if n in (which, "log_decay") or (which == "all" and n != "log_decay"):
            if n != "log_decay":
                f = 10.0 ** (low + (high - low) * torch.rand(75, 2, generator=g))
                x[i] = x[i] * (f if n == "beta" else f[..., None]).cuda()
    _run(torch, ctx, x, [75], _state(torch, 1, 2, 128), getattr(torch, kind))


@pytest.mark.parametrize("which", ["q", "k", "v", "beta"])
@pytest.mark.parametrize("size", [1e10, 1e-10, 0.0])
@pytest.mark.parametrize("at", [15, 31, 36])
def test_one_token_of_another_size(torch, ctx, which, size, at):
    """The tokens before it, in its chunk too, keep their accuracy."""
    x = _inputs(torch, 37, 2, 128, 19)
    x[NAMES.index(which)][at] *= size
    _run(torch, ctx, x, [37], _state(torch, 1, 2, 128))


@pytest.mark.parametrize("at", [0, 1, 24, 31])
def test_content_that_is_forgotten_at_once(torch, ctx, at):
    """A token that empties every channel after contents of 1e9, and small ones behind it."""
    x = _inputs(torch, 45, 2, 128, 21)
    x[3][at] = -60.0
    x[2][at:] *= 1e-3
    x[2][:at] *= 1e6
    _run(torch, ctx, x, [45], 1e9 * _state(torch, 1, 2, 128))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which,at,col", [("q", 9, 3), ("k", 9, 100), ("v", 9, 64), ("beta", 9, 0), ("log_decay", 9, 77), ("v", 31, 0),
                                          ("k", 15, 0), ("k", 0, 5), ("v", 0, 127), ("log_decay", 16, 2), ("q", 34, 8)])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_infinities_and_nan_reach_later_tokens_only(torch, ctx, bad, which, at, col, kind):
    if which == "log_decay" and bad == -math.inf:
        bad = 1e30   # exp gives infinity; -inf is a decay of zero
    dtype = getattr(torch, kind)
    x = _inputs(torch, 35, 2, 128, 23)
    state = _state(torch, 1, 2, 128)
    clean, _ = _prefill(torch, ctx, x, [35], state, dtype)
    i = NAMES.index(which)
    if which == "beta":
        x[i][at, 0] = bad
    else:
        x[i][at, 0, col] = bad
    out, new = _run(torch, ctx, x, [35], state, dtype)
    assert torch.equal(out[:at], clean[:at])
    assert torch.equal(out[:, 1], clean[:, 1]), "the other head"


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_state_rows_do_not_mix(torch, ctx, bad):
    x = _inputs(torch, 40, 1, 128, 29)
    state = _state(torch, 1, 1, 128)
    state[0, 0, 17, 99] = bad
    _run(torch, ctx, x, [40], state)


def test_one_head_or_sequence_of_another_size(torch, ctx):
    x = _inputs(torch, 100, 3, 64, 31)
    state = _state(torch, 2, 3, 64)
    x[2][:, 1] *= 1e-9
    state[:, 1] *= 1e-9
    x[2][:60] *= 1e7
    state[0] *= 1e7
    _run(torch, ctx, x, [60, 40], state)


@pytest.mark.parametrize("kept", [True, False])
def test_segments_row_by_row(torch, ctx, kept):
    """Chunk operands in more than one segment (512 heads: 70 chunks at a time), each head's and token's row on its own."""
    lengths, h, d = [613, 5, 560], 512, 128
    x = _inputs(torch, sum(lengths), h, d, 37)
    x = [t.to(torch.bfloat16).float() if i < 3 else t for i, t in enumerate(x)]
    state = _state(torch, 3, h, d)
    T = sum(lengths)
    flat = [t.reshape(T, h * d) for t in x[:4]]
    flat[:3] = [t.to(torch.bfloat16) for t in flat[:3]]
    off = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32).cuda()
    out = torch.empty(T, h * d, dtype=torch.bfloat16, device="cuda")
    new = torch.empty_like(state) if kept else None
    ctx.kda_prefill(*flat, x[4], off, out, state=state, state_out=new)
    ctx.sync()
    first = 0
    for s, n in enumerate(lengths):
        for h0 in range(0, h, 128):
            part = [t[first:first + n, h0:h0 + 128] for t in x]
            o, st, size, R = _rule(torch, part, state[s, h0:h0 + 128])
            _check(torch, out.view(T, h, d)[first:first + n, h0:h0 + 128], o, size, f"sequence {s}, heads {h0}", "out")
            if kept:
                _check(torch, new[s, h0:h0 + 128], st, R, f"state {s}, heads {h0}", "state")
        first += n


@pytest.mark.parametrize("lengths", [[300] + [1] * 16, [1] * 20 + [130] + [3] * 9 + [8, 9, 0, 7], [0, 5, 0, 200] * 8, [(7 * i) % 40 for i in range(33)],
                                     [(11 * i) % 29 for i in range(1100)]], ids=["one long first", "one long between", "with empty ones", "33", "1100"])
@pytest.mark.parametrize("d,h", [(32, 1), (128, 2)])
def test_long_and_short_sequences_together(torch, ctx, lengths, d, h):
    """Some go token by token, some in chunks; the chunks are found in the offsets."""
    if len(lengths) > 1000 and d == 128:
        lengths = lengths[:100]
    x = _inputs(torch, sum(lengths), h, d, 41 + len(lengths))
    _run(torch, ctx, x, lengths, _state(torch, len(lengths), h, d))


@pytest.mark.parametrize("at", [15, 30])
def test_a_small_state_before_a_large_value(torch, ctx, at):
    """Contents of 1e-20 are read out exactly up to the token that brings 1e12."""
    x = _inputs(torch, 40, 2, 128, 43)
    x[2][:at] *= 1e-20
    x[2][at] *= 1e12
    _run(torch, ctx, x, [40], 1e-20 * _state(torch, 1, 2, 128))


@pytest.mark.parametrize("at", [0, 14, 15])
def test_a_zero_key_beside_small_contents(torch, ctx, at):
    """A token without a key writes nothing, however large its value is."""
    x = _inputs(torch, 20, 2, 128, 47)
    x[2] *= 1e-9
    x[2][at] *= 1e21
    x[1][at] = 0.0
    _run(torch, ctx, x, [20], 1e-9 * _state(torch, 1, 2, 128))


@pytest.mark.parametrize("lengths", [[90], [100] + [1] * 20 + [30]], ids=["chunks", "tokens and chunks"])
def test_in_a_graph(torch, ctx, lengths):
    """A captured call, replayed on other inputs and other lengths."""
    T, h, d, S = sum(lengths), 2, 128, len(lengths)
    x, other = _inputs(torch, T, h, d, 53), _inputs(torch, T, h, d, 54)
    state = _state(torch, S, h, d)
    want, want_new = _prefill(torch, ctx, other, lengths[::-1], state)
    flat = [t.reshape(T, h * d).contiguous() for t in x[:4]] + [x[4]]
    off = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32).cuda()
    out, new = torch.empty(T, h * d, device="cuda"), torch.empty_like(state)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.use_stream(side)
        try:
            ctx.kda_prefill(*flat, off, out, state=state, state_out=new)
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                ctx.kda_prefill(*flat, off, out, state=state, state_out=new)
        finally:
            ctx.use_stream()
    for t, o in zip(flat, other):
        t.copy_(o.reshape(t.shape))
    off.copy_(torch.tensor(np.cumsum([0, *lengths[::-1]]), dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(T, h, d), want) and torch.equal(new, want_new)
