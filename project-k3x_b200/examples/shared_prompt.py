"""A batch of sequences that begin with one prompt, drafted and verified: the
prompt operators next to the acceptance calls.

    python project-k3x_b200/examples/shared_prompt.py [--prompt 2000] [--sequences 8] [--drafts 4] [--rounds 3]

One layer of each kind of token mixer, with random weights: the gated delta
rule (its state) and attention (its cache). The prompt goes in once:
k3xb_kda_prefill makes the state that every sequence starts from, and the
prompt's key and value rows become the shared prefix. A round then verifies
the anchor and the drafts of every sequence at once, k3xb_kda_tree for the
rule and k3xb_prefix_attention for the prefix, the sequence's own rows and the
drafts themselves, greedily accepts (k3xb_accept_greedy) and commits: the
state with k3xb_kda_commit, the cache by its length alone, since a linear
draft's rows already stand in their places. At the end one plain decode step
(k3xb_kda_step, and one node of attention) continues from what was committed,
and the whole is compared with a prefill of every sequence's full text.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import k3xb  # noqa: E402

HEADS, DIM, EXTRA, VOCAB, WIDTH = 4, 128, 64, 512, 256


class Mixers:
    """Per-token inputs of both mixers, from one embedding table."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") / cols ** 0.5).to(torch.bfloat16)

        p = HEADS * DIM
        self.embedding = torch.randn(VOCAB, WIDTH, generator=g, device="cuda").to(torch.bfloat16).float()
        self.names = {"kq": p, "kk": p, "kv": p, "decay": p, "aq": HEADS * (DIM + EXTRA), "ak": p, "av": p, "ae": EXTRA}
        self.weights = {n: weight(rows, WIDTH) for n, rows in self.names.items()}
        self.beta, self.head = weight(8, WIDTH), weight(VOCAB, 2 * p)   # 8 rows: the linear call's granularity

    def rows(self, ctx, tokens):
        """Every projection of a flat list of tokens."""
        x = self.embedding[tokens]

        def linear(w):
            out = torch.empty(x.shape[0], w.shape[0], device="cuda")
            ctx.linear_bf16(x, w, out)
            return out

        r = {n: linear(w) for n, w in self.weights.items()}
        for n in ("kq", "kk"):
            y = r[n].view(-1, HEADS, DIM)
            r[n] = (y / y.norm(dim=-1, keepdim=True)).reshape(-1, HEADS * DIM)
        r["decay"] = -5.0 * torch.sigmoid(r["decay"] - 3.0)
        r["beta"] = torch.sigmoid(linear(self.beta)[:, :HEADS]).contiguous()
        for n in ("aq", "ak", "av", "ae"):
            r[n] = r[n].to(torch.bfloat16)
        return r

    def logits(self, ctx, rule_out, attention_out):
        x = torch.cat([rule_out.reshape(-1, HEADS * DIM), attention_out.float().reshape(-1, HEADS * DIM)], dim=1)
        out = torch.empty(x.shape[0], VOCAB, device="cuda")
        ctx.linear_bf16(x.contiguous(), self.head, out, round_output=False)
        return out


def prefill(ctx, m, tokens):
    """A text by itself: its state, and its logits at every position (the
    attention as a chain of single tokens over the text's own rows)."""
    r, n = m.rows(ctx, tokens), len(tokens)
    state, out = torch.empty(1, HEADS, DIM, DIM, device="cuda"), torch.empty(n, HEADS * DIM, device="cuda")
    offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    ctx.kda_prefill(r["kq"], r["kk"], r["kv"], r["decay"], r["beta"], offsets, out, state_out=state)
    k, v, e = r["ak"].view(1, n, HEADS, DIM), r["av"].view(1, n, HEADS, DIM), r["ae"].view(1, n, EXTRA)
    att = torch.empty(n, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    # position i is a sequence of its own with i committed rows of one cache
    ctx.prefix_attention(r["aq"].view(n, 1, HEADS, DIM + EXTRA), None, None, *(t.expand(n, *t.shape[1:]) for t in (k, v)),
                         torch.arange(n, dtype=torch.int32, device="cuda"), [-1], att.view(n, 1, HEADS, DIM),
                         suffix_extra=e.expand(n, n, EXTRA))
    return state, m.logits(ctx, out, att)


def main(prompt=2000, sequences=8, drafts=4, rounds=3, seed=1):
    ctx = k3xb.Context(torch.cuda.current_device())
    ctx.use_stream()
    m, S, N = Mixers(seed), sequences, drafts + 1
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    text = torch.randint(VOCAB, (prompt,), generator=g, device="cuda")
    # the prompt, once
    r = m.rows(ctx, text)
    one = torch.empty(1, HEADS, DIM, DIM, device="cuda")
    out = torch.empty(prompt, HEADS * DIM, device="cuda")
    ctx.kda_prefill(r["kq"], r["kk"], r["kv"], r["decay"], r["beta"],
                    torch.tensor([0, prompt], dtype=torch.int32, device="cuda"), out, state_out=one)
    prefix = dict(prefix_k=r["ak"].view(prompt, HEADS, DIM), prefix_v=r["av"].view(prompt, HEADS, DIM), prefix_extra=r["ae"])
    # every sequence's state and cache
    state = one.expand(S, -1, -1, -1).contiguous()
    room = rounds * N + N + 1
    cache = dict(suffix_k=torch.zeros(S, room, HEADS, DIM, dtype=torch.bfloat16, device="cuda"),
                 suffix_v=torch.zeros(S, room, HEADS, DIM, dtype=torch.bfloat16, device="cuda"),
                 suffix_extra=torch.zeros(S, room, EXTRA, dtype=torch.bfloat16, device="cuda"))
    length = torch.zeros(S, dtype=torch.int32, device="cuda")

    def attend(r, n):
        """Stores the rows of n nodes behind each sequence's own and attends."""
        at = length.long()[:, None] + torch.arange(n, device="cuda")
        who = torch.arange(S, device="cuda")[:, None]
        for name, x in (("suffix_k", "ak"), ("suffix_v", "av"), ("suffix_extra", "ae")):
            cache[name][who, at] = r[x].view(S, n, *cache[name].shape[2:])
        att = torch.empty(S, n, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        ctx.prefix_attention(r["aq"].view(S, n, HEADS, DIM + EXTRA), prefix["prefix_k"], prefix["prefix_v"], cache["suffix_k"],
                             cache["suffix_v"], length, [i - 1 for i in range(n)], att, prefix_extra=prefix["prefix_extra"],
                             suffix_extra=cache["suffix_extra"])
        return att

    committed = [[] for _ in range(S)]
    anchor = torch.randint(VOCAB, (S,), generator=g, device="cuda")
    guess = None
    for _ in range(rounds):
        draft = torch.randint(VOCAB, (S, drafts), generator=g, device="cuda")
        if guess is not None:   # a drafter that knows the first token
            draft[:, 0] = guess
        nodes = torch.cat([anchor[:, None], draft], dim=1)
        r = m.rows(ctx, nodes.reshape(-1))
        x = [r[n].view(S, N, -1) for n in ("kq", "kk", "kv", "decay", "beta")]
        parent = [i - 1 for i in range(N)]
        rule = torch.empty(S, N, HEADS * DIM, device="cuda")
        ctx.kda_tree(state, parent, *x, rule)
        logits = m.logits(ctx, rule, attend(r, N)).view(S, N, VOCAB)
        accepted = torch.empty(S, dtype=torch.int32, device="cuda")
        tokens, count = torch.empty(S, N, dtype=torch.int32, device="cuda"), torch.empty(S, dtype=torch.int32, device="cuda")
        ctx.accept_greedy(logits, draft.to(torch.int32), accepted, tokens, count)
        ctx.sync()
        kept = accepted.tolist()
        new = torch.empty_like(state)
        ctx.kda_commit(state, parent, *x, kept, new)
        state = new
        length += accepted + 1
        for s in range(S):
            committed[s] += nodes[s, :kept[s] + 1].tolist()
        anchor = tokens[torch.arange(S, device="cuda"), accepted.long()].long()
        guess = logits[:, 0].argmax(dim=-1) if drafts else None
    # one plain step of decoding
    r = m.rows(ctx, anchor)
    rule = torch.empty(S, HEADS * DIM, device="cuda")
    ctx.kda_step(r["kq"], r["kk"], r["kv"], r["decay"], r["beta"], state, rule)
    logits = m.logits(ctx, rule, attend(r, 1))
    ctx.sync()
    # against every text on its own
    worst_state = worst_logits = 0.0
    for s in range(S):
        whole = torch.cat([text, torch.tensor(committed[s] + [int(anchor[s])], device="cuda")])
        want_state, want = prefill(ctx, m, whole)
        ctx.sync()
        worst_state = max(worst_state, float((state[s] - want_state[0]).norm() / want_state.norm()))
        worst_logits = max(worst_logits, float((logits[s] - want[-1]).abs().max() / want[-1].abs().max()))
    total = sum(len(c) for c in committed)
    ctx.close()
    return dict(prompt=prompt, sequences=S, committed=total, state_error=worst_state, logits_error=worst_logits)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("prompt", 2000), ("sequences", 8), ("drafts", 4), ("rounds", 3)):
        ap.add_argument("--" + name, type=int, default=value)
    print(main(**vars(ap.parse_args())))
