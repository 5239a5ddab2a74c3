"""Timed cases of the prompt and shared-prefix operators.

Three operators serve a batch of sequences that begin with the same long
prompt, next to the verify step:

* ``kda_prefill``: the gated delta rule over whole prompts (ragged, packed),
* ``kda_step``: the same rule for one token of each sequence, state in place,
* ``prefix_attention``: attention of draft nodes over a shared prefix, each
  sequence's own suffix and the node's ancestors in the draft topology.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, with the library's entry points. ``exact`` restates them in
64 bits, token by token and sequence by sequence.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_CTX = []

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GATE_LOWER_BOUND = -5.0   # log-decays of the KDA gate lie in (-5, 0)
CHUNK = 32                # tokens per chunk of the plain prefill


def _context():
    """The program's context, made once."""
    if not _CTX:
        pkg = os.path.join(ROOT, "project-k3x_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import k3xb
        ctx = k3xb.Context(torch.cuda.current_device())
        ctx.use_stream()
        _CTX.append(ctx)
    return _CTX[0]


# ---- cases --------------------------------------------------------------------


def listed():
    pre = dict(op="kda_prefill", heads=32, dim=128, type="f32", carried=False, fused=False, spread=3)
    step = dict(op="kda_step", heads=32, dim=128, type="f32", pool=0, idle=0)
    att = dict(op="prefix_attention", heads=32, kv_heads=32, main=128, extra=64, value=128, type="bf16", nodes=1,
               topology="chain", prefix=0, suffix=0, idle=0)
    return [
        # one long prompt goes in: every head of one sequence, a chain over the whole length
        dict(pre, name="prefill one prompt 8192", sequences=1, tokens=8192),
        # several users' turns of unlike lengths appended to states that they already have,
        # q, k and v as column slices of one projection
        dict(pre, name="prefill 13 ragged turns bf16", sequences=13, tokens=12345, type="bf16", carried=True, fused=True),
        # tool results and short turns: a few dozen tokens each, head width 64
        dict(pre, name="prefill 7 short turns d64", sequences=7, tokens=301, heads=8, dim=64, carried=True),
        # decoding one sequence: latency alone
        dict(step, name="step 1 sequence", sequences=1),
        # the decode batch of the verify stack's 64 sequences
        dict(step, name="step 64 sequences", sequences=64),
        # a large serving batch out of a pool of states with slots of its own order, some of them idle
        dict(step, name="step 333 of a pool bf16", sequences=333, type="bf16", pool=400, idle=21),
        # one user's next token after a short prompt: latency alone
        dict(att, name="attend 1 token after 700", sequences=1, prefix=700, suffix=45),
        # 64 sequences' next tokens after one long prompt and some turns of their own
        dict(att, name="attend 64 tokens after 16384", sequences=64, prefix=16384, suffix=200),
        # the verify step's shape: anchor and 8 drafts for each of 64 sequences
        dict(att, name="attend 64 x 9 drafts after 16384", sequences=64, nodes=9, prefix=16384, suffix=200, idle=3),
        # draft trees of 32 nodes, depth 4, from a 1024-token prefix
        dict(att, name="attend 6 trees of 32 f16", sequences=6, nodes=32, topology="tree", prefix=1024, suffix=77,
             type="f16"),
        # grouped heads without a shared key part, odd lengths
        dict(att, name="attend grouped heads 21 x 5", sequences=21, nodes=5, heads=32, kv_heads=4, extra=0, prefix=5003,
             suffix=331),
        # no shared prompt: every sequence reads its own rows alone
        dict(att, name="attend own rows only d64", sequences=48, heads=16, kv_heads=16, main=64, extra=0, value=64,
             suffix=2100),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["kda_prefill", "kda_step", "prefix_attention", "prefix_attention"])
    if op == "kda_prefill":
        sequences = _log_int(rng, 1, 40)
        return dict(op=op, heads=rng.choice([4, 8, 16, 32]), dim=rng.choice([64, 128, 128]), type=rng.choice(["f32", "bf16"]),
                    carried=rng.random() < 0.5, fused=rng.random() < 0.5, spread=rng.choice([1, 3, 30]),
                    sequences=sequences, tokens=max(sequences, _log_int(rng, 1, 8192)))
    if op == "kda_step":
        sequences = _log_int(rng, 1, 333)
        pool = rng.choice([0, sequences + rng.randint(1, 50)])
        return dict(op=op, heads=rng.choice([4, 8, 16, 32]), dim=rng.choice([32, 64, 128]), type=rng.choice(["f32", "bf16"]),
                    sequences=sequences, pool=pool, idle=rng.randint(0, (sequences - 1) // 4) if pool else 0)
    heads, group = rng.choice([8, 16, 32]), rng.choice([1, 1, 2, 4, 8])
    nodes = rng.choice([1, 1, 2, 3, 5, 9, 17, 32])
    sequences = _log_int(rng, 1, max(1, min(64, 600 // nodes)))
    main, extra, value = rng.choice([(128, 64, 128), (128, 0, 128), (64, 0, 64), (64, 64, 64), (128, 64, 64)])
    return dict(op=op, heads=heads, kv_heads=heads // group, main=main, extra=extra, value=value,
                type=rng.choice(["bf16", "bf16", "f16"]), nodes=nodes, topology=rng.choice(["chain", "tree"]),
                prefix=rng.choice([0, _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)]),
                suffix=rng.choice([0, _log_int(rng, 1, 700)]), sequences=sequences, idle=rng.randint(0, sequences // 8))


def _lengths(case):
    """Token counts of the prompts: `tokens` in all, the longest about `spread` times the mean or more."""
    n, total = case["sequences"], case["tokens"]
    weights = [1.0 + (case["spread"] - 1.0) * ((i * 7 + 3) % n / max(1, n - 1)) ** 2 for i in range(n)]
    lengths = [max(1, int(total * w / sum(weights))) for w in weights]
    while sum(lengths) > total and max(lengths) > 1:
        lengths[lengths.index(max(lengths))] -= min(sum(lengths) - total, max(lengths) - 1)
    lengths[lengths.index(max(lengths))] += max(0, total - sum(lengths))
    return lengths


def _parent(case):
    n = case["nodes"]
    if case["topology"] == "chain":
        return [i - 1 for i in range(n)]
    return [-1 if i == 0 else (i - 1) // 2 if i < 15 else i - 8 for i in range(n)]


def _suffix_lengths(case):
    """Each sequence's own committed rows, 0 to `suffix`; -1 where it is idle."""
    n, most = case["sequences"], case["suffix"]
    own_rows = [most if n == 1 else round(most * ((i * 5 + 2) % n) / (n - 1)) for i in range(n)]
    for i in range(case["idle"]):
        own_rows[(3 + 7 * i) % n] = -1
    return own_rows


def work(case):
    el = TYPES[case["type"]].itemsize
    if case["op"] in ("kda_prefill", "kda_step"):
        h, d = case["heads"], case["dim"]
        tokens = case["tokens"] if case["op"] == "kda_prefill" else case["sequences"] - case["idle"]
        states = case["sequences"] if case["op"] == "kda_prefill" else tokens
        reads = 1 if case["op"] == "kda_step" or case["carried"] else 0
        return {"bytes": tokens * h * (d * (4 * el + 4) + 4) + states * h * d * d * 4 * (1 + reads),
                "flops": 7.0 * tokens * h * d * d}
    rows = [n for n in _suffix_lengths(case) if n >= 0]
    n, parent = case["nodes"], _parent(case)
    depth = [0] * n
    for i in range(n):
        depth[i] = 1 + (depth[parent[i]] if parent[i] >= 0 else 0)
    keys = sum(n * (case["prefix"] + s) + sum(depth) for s in rows)
    width = case["main"] + case["extra"] + case["value"]
    per_row = el * (case["kv_heads"] * (case["main"] + case["value"]) + case["extra"])
    return {"bytes": per_row * (case["prefix"] + sum(s + n for s in rows))
            + len(rows) * n * case["heads"] * (el * width + 4),
            "flops": 2.0 * keys * case["heads"] * width}


# ---- inputs -------------------------------------------------------------------


def _gates(gen, tokens, h, d):
    """Log-decays as the KDA gate makes them (slow channels and fast ones) and write strengths."""
    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    bias = -3.0 + 2.0 * normal(1, h * d)
    log_decay = GATE_LOWER_BOUND * torch.sigmoid(bias + normal(tokens, h * d))
    return log_decay, torch.sigmoid(normal(tokens, h))


def _qkv(gen, tokens, h, d, dtype, fused):
    """Normalised queries (times 1/sqrt(d)) and keys with a part in common, and values, bf16-valued as the block makes them."""
    x = torch.randn(3, tokens, h, d, generator=gen, device="cuda")
    common = torch.randn(1, h, d, generator=gen, device="cuda")
    q, k = (x[i] + 0.5 * common for i in (0, 1))
    q = q / q.norm(dim=-1, keepdim=True) / math.sqrt(d)
    k = k / k.norm(dim=-1, keepdim=True)
    flat = [t.to(torch.bfloat16).to(dtype).reshape(tokens, h * d) for t in (q, k, x[2])]
    if fused:
        flat = list(torch.cat(flat, dim=1).split(h * d, dim=1))
    return flat


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    dtype = TYPES[case["type"]]
    st = dict(case)
    if case["op"] == "kda_prefill":
        n, total, h, d = case["sequences"], case["tokens"], case["heads"], case["dim"]
        lengths = _lengths(case)
        offsets = [0]
        for x in lengths:
            offsets.append(offsets[-1] + x)
        q, k, v = _qkv(gen, total, h, d, dtype, case["fused"])
        log_decay, beta = _gates(gen, total, h, d)
        st.update(q=q, k=k, v=v, log_decay=log_decay, beta=beta, state=0.3 * normal(n, h, d, d) if case["carried"] else None,
                  state_out=torch.empty(n, h, d, d, device="cuda"), out=torch.empty(total, h * d, dtype=dtype, device="cuda"),
                  offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), lengths=lengths)
        st.update(_chunk_plan(lengths, offsets))
        return st
    if case["op"] == "kda_step":
        n, h, d = case["sequences"], case["heads"], case["dim"]
        q, k, v = _qkv(gen, n, h, d, dtype, False)
        log_decay, beta = _gates(gen, n, h, d)
        slots = None
        if case["pool"]:
            slots = torch.randperm(case["pool"], generator=gen, device="cuda")[:n].to(torch.int32)
            slots[[(1 + 3 * i) % n for i in range(case["idle"])]] = -1
        st.update(q=q, k=k, v=v, log_decay=log_decay, beta=beta, state=0.3 * normal(case["pool"] or n, h, d, d), slots=slots,
                  out=torch.empty(n, h * d, dtype=dtype, device="cuda"))
        return st
    n, nodes, heads, kvh = case["sequences"], case["nodes"], case["heads"], case["kv_heads"]
    main, extra, value, prefix = case["main"], case["extra"], case["value"], case["prefix"]
    parent = _parent(case)
    capacity = case["suffix"] + nodes + 3   # rows past a sequence's own hold what earlier turns left there
    st.update(q=(2.0 * normal(n, nodes, heads, main + extra)).to(dtype), parent=parent,
              prefix_k=normal(prefix, kvh, main).to(dtype), prefix_v=normal(prefix, kvh, value).to(dtype),
              prefix_extra=normal(prefix, extra).to(dtype) if extra else None,
              suffix_k=normal(n, capacity, kvh, main).to(dtype), suffix_v=normal(n, capacity, kvh, value).to(dtype),
              suffix_extra=normal(n, capacity, extra).to(dtype) if extra else None,
              suffix_len=torch.tensor(_suffix_lengths(case), dtype=torch.int32, device="cuda"),
              out=torch.empty(n, nodes, heads, value, dtype=dtype, device="cuda"),
              lse=torch.empty(n, nodes, heads, device="cuda"))
    if prefix:
        st["prefix_k"][0] *= 2.0   # the first position draws attention
    sees = torch.zeros(nodes, nodes, dtype=torch.bool)
    for i in range(nodes):
        j = i
        while j >= 0:
            sees[i, j] = True
            j = parent[j]
    st["sees"] = sees.cuda()
    return st


def _chunk_plan(lengths, offsets):
    """Chunks of the plain prefill: the tokens of each (-1: none), and, chunk by chunk, the sequences that reach it."""
    by_length = sorted(range(len(lengths)), key=lambda s: -lengths[s])
    tokens, steps = [], []
    for c in range((max(lengths) + CHUNK - 1) // CHUNK):
        here = [s for s in by_length if lengths[s] > c * CHUNK]
        steps.append((len(tokens), len(here)))
        for s in here:
            first = c * CHUNK
            tokens.append([offsets[s] + first + i if first + i < lengths[s] else -1 for i in range(CHUNK)])
    return dict(chunk_tokens=torch.tensor(tokens, device="cuda"), chunk_steps=steps,
                by_length=torch.tensor(by_length, device="cuda"))


# ---- one pass -----------------------------------------------------------------


def run(state):
    s = state
    if own:
        ctx = _context()
        if s["op"] == "kda_prefill":
            ctx.kda_prefill(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["offsets"], s["out"], state=s["state"],
                            state_out=s["state_out"])
            return s["out"], s["state_out"]
        if s["op"] == "kda_step":
            ctx.kda_step(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], s["out"], slots=s["slots"])
            return s["out"], s["state"]
        ctx.prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["suffix_k"], s["suffix_v"], s["suffix_len"],
                             s["parent"], s["out"], prefix_extra=s["prefix_extra"], suffix_extra=s["suffix_extra"],
                             lse=s["lse"])
        return s["out"], s["lse"]
    return {"kda_prefill": _plain_prefill, "kda_step": _plain_step, "prefix_attention": _plain_attention}[s["op"]](s)


def _plain_prefill(s):
    h, d = s["heads"], s["dim"]
    at = s["chunk_tokens"]
    live = (at >= 0)[:, :, None]
    at = at.clamp(min=0)

    def chunks(x, width):   # [chunks, h, CHUNK, width] in 32 bits, zero where a chunk has no token
        return (x[at].float() * live).view(len(at), CHUNK, h, width).transpose(1, 2).contiguous()

    q, k, v = (chunks(s[n], d) for n in ("q", "k", "v"))
    decay = chunks(s["log_decay"], d).cumsum(dim=2)
    beta = chunks(s["beta"], 1)
    # products of rows i and j with the decay between them, for j <= i
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    kk, qk = (torch.empty(len(at), h, CHUNK, CHUNK, device="cuda") for _ in range(2))
    part = max(1, (1 << 28) // (h * CHUNK * CHUNK * d))
    for c in range(0, len(at), part):
        w = slice(c, c + part)
        between = decay[w, :, :, None, :] - decay[w, :, None, :, :]
        keys = torch.exp(between.masked_fill(~lower[:, :, None], -math.inf)) * k[w, :, None, :, :]
        kk[w] = (keys @ k[w, :, :, :, None])[..., 0]
        qk[w] = (keys @ q[w, :, :, :, None])[..., 0]
    # (1 + m)^-1 for the strictly lower m = beta kk: its powers from CHUNK on are zero
    m = beta * kk.masked_fill(~lower.tril(-1), 0.0)
    inverse, power = torch.eye(CHUNK, device="cuda") - m, m @ m
    for _ in range(4):
        inverse, power = inverse + inverse @ power, power @ power
    from_start, to_end = torch.exp(decay), torch.exp(decay[:, :, -1:] - decay)
    w = inverse @ (beta * k * from_start)
    u = inverse @ (beta * v)
    qs, ks = q * from_start, k * to_end
    n = s["sequences"]
    state = s["state"][s["by_length"]] if s["state"] is not None else torch.zeros(n, h, d, d, device="cuda")
    o = torch.empty_like(v)
    for first, count in s["chunk_steps"]:
        c, now = slice(first, first + count), state[:count]
        delta = u[c] - w[c] @ now.transpose(2, 3)
        o[c] = qs[c] @ now.transpose(2, 3) + qk[c] @ delta
        state[:count] = now * from_start[c, :, -1:] + delta.transpose(2, 3) @ ks[c]
    s["out"][at[live[:, :, 0]]] = o.transpose(1, 2).reshape(len(at), CHUNK, h * d)[live[:, :, 0]].to(s["out"].dtype)
    s["state_out"][s["by_length"]] = state
    return s["out"], s["state_out"]


def _plain_step(s):
    n, h, d = s["sequences"], s["heads"], s["dim"]
    q, k, v, log_decay = (s[x].float().view(n, h, d) for x in ("q", "k", "v", "log_decay"))
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(n, device="cuda")
    live = slots >= 0
    state = s["state"][slots.clamp(min=0)] * torch.exp(log_decay)[:, :, None, :]
    delta = (v - (state @ k[..., None])[..., 0]) * s["beta"][:, :, None]
    state = state + delta[..., None] * k[:, :, None, :]
    out = (state @ q[..., None])[..., 0] * live[:, None, None]
    s["out"].copy_(out.view(n, h * d))
    s["state"][slots[live]] = state[live]
    return s["out"], s["state"]


def _plain_attention(s):
    n, nodes, heads, kvh, value, prefix = (s[x] for x in ("sequences", "nodes", "heads", "kv_heads", "value", "prefix"))
    g = heads // kvh
    width = s["main"] + s["extra"]

    def keys(k, extra):   # every head's key, its part of the shared one behind its own
        k = k.float()
        return k if extra is None else torch.cat([k, extra.float().unsqueeze(-2).expand(*k.shape[:-1], s["extra"])], dim=-1)

    q = s["q"].float().view(n, nodes, kvh, g, width) / math.sqrt(width)
    by_head = q.permute(2, 0, 1, 3, 4).reshape(kvh, n * nodes * g, width)
    shared = by_head @ keys(s["prefix_k"], s["prefix_extra"]).permute(1, 2, 0)
    shared = shared.view(kvh, n, nodes * g, prefix)
    mine = q.permute(2, 0, 1, 3, 4).reshape(kvh, n, nodes * g, width) @ keys(s["suffix_k"], s["suffix_extra"]).permute(2, 0, 3, 1)
    row = torch.arange(s["suffix_k"].shape[1], device="cuda")
    node = row - s["suffix_len"][:, None]
    of_tree = s["sees"][:, node.clamp(0, nodes - 1)].permute(1, 0, 2) & ((node >= 0) & (node < nodes))[:, None, :]
    live = (s["suffix_len"] >= 0)[:, None, None]
    sees = ((node < 0)[:, None, :] | of_tree) & live
    mine = mine.view(kvh, n, nodes, g, -1).masked_fill(~sees[None, :, :, None, :], -math.inf).view(kvh, n, nodes * g, -1)
    shared = shared.masked_fill(~live, -math.inf)
    top = mine.amax(dim=-1, keepdim=True)
    if prefix:
        top = torch.maximum(top, shared.amax(dim=-1, keepdim=True))
    base = top.masked_fill(top == -math.inf, 0.0)
    shared, mine = torch.exp(shared - base), torch.exp(mine - base)
    total = shared.sum(dim=-1, keepdim=True) + mine.sum(dim=-1, keepdim=True)
    out = (shared.view(kvh, n * nodes * g, prefix) @ s["prefix_v"].float().transpose(0, 1)).view(kvh, n, nodes * g, value)
    out = (out + mine @ s["suffix_v"].float().permute(2, 0, 1, 3)) / total.masked_fill(total == 0.0, 1.0)
    s["out"].copy_(out.view(kvh, n, nodes, g, value).permute(1, 2, 0, 3, 4).reshape(n, nodes, heads, value))
    s["lse"].copy_((top + torch.log(total)).view(kvh, n, nodes, g).permute(1, 2, 0, 3).reshape(n, nodes, heads))
    return s["out"], s["lse"]


# ---- the definitions in 64 bits -------------------------------------------------


def _rule(state, q, k, v, log_decay, beta):
    """The gated delta rule for one token of each head: state [.., value, key]."""
    state = state * log_decay.exp().unsqueeze(-2)
    missing = v - torch.einsum("...vk,...k->...v", state, k)
    state = state + torch.einsum("...v,...k->...vk", missing * beta.unsqueeze(-1), k)
    return state, torch.einsum("...vk,...k->...v", state, q)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "kda_prefill":
        h, d = case["heads"], case["dim"]
        lengths, first = s["lengths"], s["offsets"].tolist()
        x = [s[n].double().view(-1, h, d) for n in ("q", "k", "v", "log_decay")] + [s["beta"].double()]
        out = torch.zeros(case["tokens"], h, d, dtype=torch.float64, device="cuda")
        state = s["state"].double() if case["carried"] else torch.zeros(len(lengths), h, d, d, dtype=torch.float64, device="cuda")
        for t in range(max(lengths)):
            who = [i for i, n in enumerate(lengths) if n > t]
            at = torch.tensor([first[i] + t for i in who], device="cuda")
            w = torch.tensor(who, device="cuda")
            new, out[at] = _rule(state[w] if len(who) < len(lengths) else state, *(y[at] for y in x))
            if len(who) < len(lengths):
                state[w] = new
            else:
                state = new
        return out.view(case["tokens"], h * d), state
    if case["op"] == "kda_step":
        n, h, d = case["sequences"], case["heads"], case["dim"]
        x = [s[m].double().view(n, h, d) for m in ("q", "k", "v", "log_decay")] + [s["beta"].double()]
        state = s["state"].double()
        out = torch.zeros(n, h, d, dtype=torch.float64, device="cuda")
        slots = s["slots"].tolist() if s["slots"] is not None else list(range(n))
        for i, slot in enumerate(slots):
            if slot >= 0:
                state[slot], out[i] = _rule(state[slot], *(y[i] for y in x))
        return out.view(n, h * d), state
    n, nodes, heads, kvh = case["sequences"], case["nodes"], case["heads"], case["kv_heads"]
    own_rows = s["suffix_len"].tolist()
    out = torch.zeros(n, nodes, heads, case["value"], dtype=torch.float64, device="cuda")
    lse = torch.full((n, nodes, heads), -math.inf, dtype=torch.float64, device="cuda")

    def per_head(x):
        return x.double().repeat_interleave(heads // kvh, dim=1)

    pk, pv = per_head(s["prefix_k"]), per_head(s["prefix_v"])
    for i in range(n):
        if own_rows[i] < 0:
            continue
        rows = own_rows[i] + nodes
        k = torch.cat([pk, per_head(s["suffix_k"][i, :rows])])
        v = torch.cat([pv, per_head(s["suffix_v"][i, :rows])])
        q = s["q"][i].double()
        logits = torch.einsum("nhd,lhd->nhl", q[..., :case["main"]], k)
        if case["extra"]:
            e = torch.cat([s["prefix_extra"], s["suffix_extra"][i, :rows]]).double()
            logits += torch.einsum("nhd,ld->nhl", q[..., case["main"]:], e)
        logits /= math.sqrt(case["main"] + case["extra"])
        for m in range(nodes):
            hidden = set(range(nodes))
            j = m
            while j >= 0:
                hidden.discard(j)
                j = s["parent"][j]
            if hidden:
                logits[m][:, [case["prefix"] + own_rows[i] + j for j in hidden]] = -math.inf
        lse[i] = torch.logsumexp(logits, dim=-1)
        out[i] = torch.einsum("nhl,lhv->nhv", torch.exp(logits - lse[i][..., None]), v)
    return out, lse
