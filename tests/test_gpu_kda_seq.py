"""The gated delta rule over whole prompts (k3xb_kda_prefill) and for one
token of each sequence (k3xb_kda_step) against the rule in 64 bits, token by
token (official_kda.cpp:319-369).

Tolerances. A sum of d <= 128 float products is off by at most 128 * 2^-24 =
7.6e-6 of its terms' size, and a token adds a few roundings of 2^-24 = 6e-8 to
a state that its decay shrinks: 1e-5 of the 2-norm for states and f32
outputs. bf16 outputs are rounded once more, by at most 2^-8 of each value.
"""
import numpy as np
import pytest

from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

TOL = 1e-5


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


def _rule(torch, q, k, v, log_decay, beta, state):
    """One sequence in 64 bits: q/k/v/log_decay [T][h][d], beta [T][h], state [h][d][d]."""
    out = torch.zeros_like(q)
    for t in range(q.shape[0]):
        state = state * log_decay[t].exp()[:, None, :]
        delta = (v[t] - (state * k[t][:, None, :]).sum(-1)) * beta[t][:, None]
        state = state + delta[:, :, None] * k[t][:, None, :]
        out[t] = (state * q[t][:, None, :]).sum(-1)
    return out, state


def _inputs(torch, T, h, d, dtype, seed, gate="mixed", unit=True):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(T, h, d, generator=g) for _ in range(3))
    if unit:
        q, k = q / q.norm(dim=-1, keepdim=True), k / k.norm(dim=-1, keepdim=True)
    if gate == "mixed":      # slow and fast channels
        ld = -5.0 * torch.sigmoid(2.0 * torch.randn(1, h, d, generator=g) - 3.0 + torch.randn(T, h, d, generator=g))
    elif gate == "none":
        ld = torch.zeros(T, h, d)
    elif gate == "strong":   # a few steps leave nothing of a channel that float can hold
        ld = -200.0 * torch.rand(T, h, d, generator=g)
    elif gate == "forget":   # exact zeros in the decay
        ld = torch.where(torch.rand(T, h, d, generator=g) < 0.1, -float("inf"), 0.0) - 0.1
    beta = torch.rand(T, h, generator=g)
    x = [t.to(dtype).cuda() for t in (q, k, v)]
    return [*(t.reshape(T, h * d) for t in x), ld.reshape(T, h * d).cuda(), beta.cuda()]


def _want(torch, x, lengths, h, d, state):
    q, k, v, ld, beta = (t.double() for t in x)
    T = q.shape[0]
    outs, states, at = [], [], 0
    for s, n in enumerate(lengths):
        w = slice(at, at + n)
        o, st = _rule(torch, *(t[w].reshape(n, h, d) for t in (q, k, v, ld)), beta[w],
                      state[s].double() if state is not None else torch.zeros(h, d, d, dtype=torch.float64, device="cuda"))
        outs.append(o.reshape(n, h * d))
        states.append(st)
        at += n
    assert at == T
    return torch.cat(outs), torch.stack(states)


def _near(torch, got, want, what, tol=TOL):
    err = float((got.double() - want).norm())
    bound = tol * float(want.norm())
    if got.dtype == torch.bfloat16:
        bound += 2.0 ** -8 * float(want.norm())
    assert np.isfinite(err) and err <= bound + 1e-30, f"{what}: 2-norm of the error {err:.3e} > {bound:.3e}"


def _prefill(torch, ctx, x, lengths, h, d, state, **kw):
    off = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32).cuda()
    out = torch.full((x[0].shape[0], h * d), 7.0, dtype=x[0].dtype, device="cuda")
    new = torch.full((len(lengths), h, d, d), 7.0, device="cuda")
    ctx.kda_prefill(*x, off, out, state=state, state_out=new, **kw)
    ctx.sync()
    return out, new


LENGTHS = [[1], [2, 0, 3], [8, 9, 7, 10, 0, 1, 30], [1] * 70 + [40], [15, 16, 17, 1], [31, 33, 64], [63, 65], [130, 0, 1, 257, 5]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("d,h", [(32, 3), (64, 2), (128, 3)])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_prefill_matches_the_rule(torch, ctx, lengths, d, h, kind):
    x = _inputs(torch, sum(lengths), h, d, getattr(torch, kind), 11 + d + len(lengths))
    g = torch.Generator().manual_seed(5)
    for state in (None, torch.randn(len(lengths), h, d, d, generator=g).cuda()):
        out, new = _prefill(torch, ctx, x, lengths, h, d, state)
        want_out, want_new = _want(torch, x, lengths, h, d, state)
        _near(torch, out, want_out, "out")
        _near(torch, new, want_new, "state")


@pytest.mark.parametrize("gate", ["none", "strong", "forget"])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_gates(torch, ctx, gate, d):
    lengths, h = [70, 33], 2
    x = _inputs(torch, sum(lengths), h, d, torch.float32, 23 + d, gate)
    state = torch.randn(2, h, d, d, generator=torch.Generator().manual_seed(6)).cuda()
    out, new = _prefill(torch, ctx, x, lengths, h, d, state)
    want_out, want_new = _want(torch, x, lengths, h, d, state)
    _near(torch, out, want_out, "out")
    _near(torch, new, want_new, "state")


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 3e5, 1e12])
def test_prefill_magnitudes(torch, ctx, scale):
    """Values and the state of any size: the rule is linear in them."""
    lengths, h, d = [50, 81], 2, 128
    x = _inputs(torch, sum(lengths), h, d, torch.float32, 31)
    x[2] = x[2] * scale
    state = scale * torch.randn(2, h, d, d, generator=torch.Generator().manual_seed(7)).cuda()
    out, new = _prefill(torch, ctx, x, lengths, h, d, state)
    want_out, want_new = _want(torch, x, lengths, h, d, state)
    _near(torch, out, want_out, "out")
    _near(torch, new, want_new, "state")


def test_prefill_large_queries_small_keys(torch, ctx):
    """Queries and keys are not normalised for the caller."""
    lengths, h, d = [47], 2, 128
    x = _inputs(torch, 47, h, d, torch.float32, 37)
    x[0], x[1] = x[0] * 3e4, x[1] * 1e-3
    out, new = _prefill(torch, ctx, x, lengths, h, d, None)
    want_out, want_new = _want(torch, x, lengths, h, d, None)
    _near(torch, out, want_out, "out")
    _near(torch, new, want_new, "state")


def test_prefill_repeated_key(torch, ctx):
    """One key over and over with beta 1: each value replaces the one before,
    so the rows of (1 + M)^-1 keep alternating signs of size 1."""
    T, h, d = 96, 2, 128
    x = _inputs(torch, T, h, d, torch.float32, 41, "none")
    x[1][:] = x[1][0]
    x[4][:] = 1.0
    out, new = _prefill(torch, ctx, x, [T], h, d, None)
    want_out, want_new = _want(torch, x, [T], h, d, None)
    _near(torch, out, want_out, "out")
    _near(torch, new, want_new, "state")


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_prefill_rows_of_one_projection(torch, ctx, kind, shift):
    """q, k and v as column slices, at rows that start at any element."""
    lengths, h, d = [40, 21], 2, 64
    dtype = getattr(torch, kind)
    x = _inputs(torch, 61, h, d, dtype, 43)
    wide = torch.zeros(61, 3 * h * d + 1 + shift, dtype=dtype, device="cuda")
    parts = [wide[:, shift + i * h * d: shift + (i + 1) * h * d] for i in range(3)]
    for p, t in zip(parts, x):
        p.copy_(t)
    out, new = _prefill(torch, ctx, [*parts, *x[3:]], lengths, h, d, None)
    ref, ref_new = _prefill(torch, ctx, x, lengths, h, d, None)
    want_out, want_new = _want(torch, x, lengths, h, d, None)
    _near(torch, out, want_out, "out")
    _near(torch, new, want_new, "state")
    assert torch.equal(out, ref) and torch.equal(new, ref_new)


def test_prefill_in_pieces_and_in_place(torch, ctx):
    """Two calls that carry the state (kept in place) give one call's result,
    and the call is deterministic."""
    h, d = 3, 128
    x = _inputs(torch, 150, h, d, torch.float32, 47)
    whole, new = _prefill(torch, ctx, x, [150], h, d, None)
    again, new2 = _prefill(torch, ctx, x, [150], h, d, None)
    assert torch.equal(whole, again) and torch.equal(new, new2)
    state = torch.zeros(1, h, d, d, device="cuda")
    out = torch.empty_like(whole)
    for a, b in ((0, 77), (77, 150)):
        off = torch.tensor([0, b - a], dtype=torch.int32).cuda()
        ctx.kda_prefill(*(t[a:b].contiguous() for t in x), off, out[a:b], state=state, state_out=state)
    ctx.sync()
    want_out, want_new = _want(torch, x, [150], h, d, None)
    _near(torch, out, want_out, "out")
    _near(torch, state, want_new, "state")


@pytest.mark.parametrize("kept", [True, False])
def test_prefill_in_segments(torch, ctx, kept):
    """More chunk operands than are held at a time (1 GiB, 72 chunks of 512
    heads): sequences begin and end in different segments, their states
    between segments in state_out or, where that is not wanted, elsewhere."""
    lengths, h, d = [700, 3, 590], 512, 128
    x = _inputs(torch, sum(lengths), h, d, torch.bfloat16, 49)
    off = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32).cuda()
    out = torch.empty(sum(lengths), h * d, dtype=torch.bfloat16, device="cuda")
    state = torch.randn(3, h, d, d, generator=torch.Generator().manual_seed(11)).cuda()
    new = torch.empty_like(state) if kept else None
    ctx.kda_prefill(*x, off, out, state=state, state_out=new)
    ctx.sync()
    want_out, want_new = _want(torch, x, lengths, h, d, state)
    _near(torch, out, want_out, "out")
    if kept:
        _near(torch, new, want_new, "state")


def test_prefill_on_another_stream(torch, ctx):
    h, d = 2, 128
    x = _inputs(torch, 90, h, d, torch.float32, 53)
    ref, _ = _prefill(torch, ctx, x, [90], h, d, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ctx.use_stream(side)
    try:
        with torch.cuda.stream(side):
            out, _ = _prefill(torch, ctx, x, [90], h, d, None)
    finally:
        ctx.use_stream()
    assert torch.equal(out, ref)


def test_prefill_agrees_with_the_tree_call(torch, ctx):
    h, d, T = 2, 128, 24
    x = _inputs(torch, T, h, d, torch.float32, 59)
    state = torch.randn(1, h, d, d, generator=torch.Generator().manual_seed(8)).cuda()
    out, _ = _prefill(torch, ctx, x, [T], h, d, state)
    tree = torch.empty(1, T, h * d, device="cuda")
    ctx.kda_tree(state, [i - 1 for i in range(T)], *(t[None] for t in x), tree)
    ctx.sync()
    _near(torch, out, tree[0].double(), "out", 2 * TOL)


def test_prefill_bad_offsets_are_reported(torch, ctx):
    import k3xb
    h, d = 2, 64
    x = _inputs(torch, 20, h, d, torch.float32, 61)
    out = torch.zeros(20, h * d, device="cuda")
    new = torch.zeros(3, h, d, d, device="cuda")
    ctx.kda_prefill(*x, torch.tensor([0, 9, 5, 21], dtype=torch.int32).cuda(), out, state_out=new)
    with pytest.raises(k3xb.K3xbError) as e:
        ctx.sync()
    assert e.value.status == k3xb.INVALID_EXTENT
    want_out, want_new = _want(torch, [t[:9] for t in x], [9], h, d, None)
    _near(torch, out[:9], want_out, "out")      # the sequence with a range is served
    _near(torch, new[:1], want_new, "state")
    assert not out[9:].any() and not new[1:].any()
    ctx.sync()


@pytest.mark.parametrize("d,h", [(32, 5), (64, 3), (128, 2)])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("S", [1, 7, 150])
def test_step_matches_the_rule(torch, ctx, d, h, kind, S):
    x = _inputs(torch, S, h, d, getattr(torch, kind), 67 + d + S)
    state = torch.randn(S, h, d, d, generator=torch.Generator().manual_seed(9)).cuda()
    want_out, want_new = _want(torch, x, [1] * S, h, d, state)
    out = torch.empty(S, h * d, dtype=x[0].dtype, device="cuda")
    ctx.kda_step(*x, state, out)
    ctx.sync()
    _near(torch, out, want_out, "out")
    _near(torch, state, want_new, "state")


def test_step_slots_and_idle_sequences(torch, ctx):
    import k3xb
    S, h, d, pool = 6, 2, 128, 11
    x = _inputs(torch, S, h, d, torch.float32, 71)
    state = torch.randn(pool, h, d, d, generator=torch.Generator().manual_seed(10)).cuda()
    before = state.clone()
    slots = [9, -1, 0, 4, -7, 10]
    out = torch.full((S, h * d), 7.0, device="cuda")
    ctx.kda_step(*x, state, out, slots=torch.tensor(slots, dtype=torch.int32).cuda())
    ctx.sync()
    live = [i for i, s in enumerate(slots) if s >= 0]
    at = [slots[i] for i in live]
    want_out, want_new = _want(torch, [t[live] for t in x], [1] * len(live), h, d, before[at])
    _near(torch, out[live], want_out, "out")
    _near(torch, state[at], want_new, "state")
    assert not out[[1, 4]].any()
    rest = [i for i in range(pool) if i not in at]
    assert torch.equal(state[rest], before[rest])
    # a slot past the pool is left out and reported
    kept = state.clone()
    ctx.kda_step(*x, state, out, slots=torch.tensor([pool, -1, -1, -1, -1, -1], dtype=torch.int32).cuda())
    with pytest.raises(k3xb.K3xbError) as e:
        ctx.sync()
    assert e.value.status == k3xb.INVALID_EXTENT and torch.equal(state, kept) and not out.any()
    ctx.sync()


def test_steps_continue_a_prefill(torch, ctx):
    h, d, T = 2, 128, 20
    x = _inputs(torch, T, h, d, torch.float32, 73)
    want_out, want_new = _want(torch, x, [T], h, d, None)
    out, state = _prefill(torch, ctx, [t[:15] for t in x], [15], h, d, None)
    _near(torch, out, want_out[:15], "prompt")
    row = torch.empty(1, h * d, device="cuda")
    for t in range(15, T):
        ctx.kda_step(*(y[t:t + 1] for y in x), state, row)
        ctx.sync()
        _near(torch, row, want_out[t:t + 1], f"token {t}")
    _near(torch, state, want_new, "state")


def test_refusals(torch, ctx):
    import k3xb
    h, d, T = 2, 64, 4
    x = _inputs(torch, T, h, d, torch.float32, 79)
    off = torch.tensor([0, T], dtype=torch.int32).cuda()
    out = torch.empty(T, h * d, device="cuda")
    state = torch.zeros(T, h, d, d, device="cuda")
    bad_state = torch.zeros(h * d * d + 1, device="cuda")[1:].view(1, h, d, d)
    odd = [torch.zeros(T, 2 * 48, device="cuda") for _ in range(4)]
    calls = [
        lambda: ctx.kda_prefill(*x, off, out, state=bad_state),                                  # unaligned state
        lambda: ctx.kda_prefill(*odd, x[4], off, torch.empty(T, 96, device="cuda")),              # head width 48
        lambda: ctx.kda_prefill(*x, off.cpu(), out),                                             # host offsets
        lambda: ctx.kda_prefill(*x, off, out.bfloat16()),                                        # out of another type
        lambda: ctx.kda_prefill(*(t.half() for t in x[:3]), *x[3:], off, out.half()),             # f16
        lambda: ctx.kda_prefill(x[0], x[1][:3], *x[2:], off, out),
        lambda: ctx.kda_prefill(*(t[:1].expand_as(t) for t in x[:3]), *x[3:], off, out),          # one row for all tokens
        lambda: ctx.kda_prefill(*x, off[:1], out),                                               # no sequence
        lambda: ctx.kda_step(*x, state[:2], out),                                                # fewer states than rows
        lambda: ctx.kda_step(*x, state.double(), out),
        lambda: ctx.kda_step(*x, state, out, slots=torch.zeros(3, dtype=torch.int32).cuda()),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(k3xb.K3xbError) as e:
            call()
        assert e.value.status == k3xb.INVALID_EXTENT, i
    lib = ctx.lib
    p = [t.data_ptr() for t in x]
    assert lib.k3xb_kda_prefill(ctx.h, p[0], p[1], p[2], h * d - 1, 0, p[3], p[4], off.data_ptr(), 1, T, h, d, None, None,
                                out.data_ptr()) == k3xb.INVALID_EXTENT
    assert lib.k3xb_kda_prefill(ctx.h, None, p[1], p[2], 0, 0, p[3], p[4], off.data_ptr(), 1, T, h, d, None, None,
                                out.data_ptr()) == k3xb.INVALID_EXTENT
    assert lib.k3xb_kda_step(ctx.h, p[0], p[1], p[2], 0, 0, p[3], p[4], T, h, d, None, T, None,
                             out.data_ptr()) == k3xb.INVALID_EXTENT
    ctx.sync()
