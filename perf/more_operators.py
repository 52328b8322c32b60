"""Grouped attention of packed prompts and of drafted trees: the calls whose speed counts, and their plain forms.

Kinds of cases and what a program uses them for:

* ``attend``: ``packed_attention`` without gradients: prompts of different
  lengths laid end to end, several query heads on one key head;
* ``train``: the same with the gradients of q, k and v;
* ``tree``: ``tree_attention``, the drafted tokens of each sequence (a tree, a
  chain, or the one next token) against its key and value cache.

With ``own`` false, ``run`` computes the operators in float32 from elementary
torch operations; ``exact`` restates them in float64.
"""

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One layer of the smallest encoder over two short prompts: launches count.
        {"name": "attend_short", "kind": "attend", "heads": 4, "kv_heads": 4, "dim": 64, "dim_v": 64, "dtype": "fp32",
         "causal": True, "seqs": 2, "tokens": 256, "mix": 1, "spare": 0, "padded": False},
        # A server's batch of prompts of different lengths, in a buffer of fixed size that they do not fill.
        {"name": "attend_prompts", "kind": "attend", "heads": 16, "kv_heads": 2, "dim": 128, "dim_v": 128,
         "dtype": "bf16", "causal": True, "seqs": 24, "tokens": 16384, "mix": 2, "spare": 512, "padded": False},
        # One long document.
        {"name": "attend_long", "kind": "attend", "heads": 8, "kv_heads": 2, "dim": 128, "dim_v": 128, "dtype": "bf16",
         "causal": True, "seqs": 1, "tokens": 32768, "mix": 3, "spare": 0, "padded": False},
        # Bidirectional encoding of many ragged texts, heads that fill no tile, values narrower than keys.
        {"name": "attend_odd", "kind": "attend", "heads": 6, "kv_heads": 3, "dim": 80, "dim_v": 48, "dtype": "fp16",
         "causal": False, "seqs": 37, "tokens": 9001, "mix": 4, "spare": 23, "padded": False},
        # A training step's attention in the smallest encoder, float32 throughout.
        {"name": "train_short", "kind": "train", "heads": 4, "kv_heads": 2, "dim": 64, "dim_v": 64, "dtype": "fp32",
         "causal": True, "seqs": 3, "tokens": 300, "mix": 5, "spare": 0, "padded": False},
        # A training step of the ordinary encoder (d_model 512): eight right-padded sequences of 1024.
        {"name": "train_padded", "kind": "train", "heads": 8, "kv_heads": 8, "dim": 64, "dim_v": 64, "dtype": "fp16",
         "causal": True, "seqs": 8, "tokens": 8192, "mix": 6, "spare": 0, "padded": True},
        # A training step over many short documents in one row of tokens.
        {"name": "train_packed", "kind": "train", "heads": 16, "kv_heads": 4, "dim": 64, "dim_v": 64, "dtype": "bf16",
         "causal": True, "seqs": 96, "tokens": 32768, "mix": 7, "spare": 0, "padded": False},
        # A training step over two long documents, wide heads.
        {"name": "train_long", "kind": "train", "heads": 16, "kv_heads": 8, "dim": 128, "dim_v": 128, "dtype": "bf16",
         "causal": True, "seqs": 2, "tokens": 16384, "mix": 8, "spare": 0, "padded": False},
        # A small tree of drafted tokens for one sequence: latency.
        {"name": "tree_one", "kind": "tree", "heads": 8, "kv_heads": 8, "dim": 64, "dim_v": 64, "dtype": "fp16",
         "batch": 1, "new": 8, "capacity": 1024, "tree": True},
        # A large tree for each of a batch of conversations, some with fewer drafts than the others.
        {"name": "tree_batch", "kind": "tree", "heads": 16, "kv_heads": 4, "dim": 128, "dim_v": 128, "dtype": "bf16",
         "batch": 16, "new": 64, "capacity": 8192, "tree": True},
        # Trees over very long caches.
        {"name": "tree_long", "kind": "tree", "heads": 16, "kv_heads": 4, "dim": 128, "dim_v": 128, "dtype": "bf16",
         "batch": 8, "new": 16, "capacity": 65536, "tree": True},
        # The next token of every sequence of a large batch, no drafts.
        {"name": "next_token", "kind": "tree", "heads": 16, "kv_heads": 4, "dim": 64, "dim_v": 64, "dtype": "fp16",
         "batch": 64, "new": 1, "capacity": 4096, "tree": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "train", "train", "train", "tree", "tree", "tree"))
    limit = max(work(c)["flops"] for c in listed() if c["kind"] == kind)
    most_bytes = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
    while True:
        dim = rng.choice((16, 32, 40, 64, 64, 64, 80, 96, 128, 128, 128))
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        case = {"kind": kind, "heads": kv_heads * rng.choice((1, 1, 2, 3, 4, 8)), "kv_heads": kv_heads, "dim": dim,
                "dim_v": rng.choice((dim, dim, dim, 64, 128)), "dtype": rng.choice(("fp32", "fp16", "fp16", "bf16", "bf16"))}
        if kind == "tree":
            case.update(batch=_log_int(rng, 1, 64), new=rng.choice((1, 1, 2, 5, 8, 16, 33, 64)),
                        capacity=_log_int(rng, 80, 65536), tree=rng.random() < 0.7)
            if work(case)["bytes"] <= most_bytes and work(case)["flops"] * _cost(case) <= limit:
                return case
            continue
        seqs = _log_int(rng, 1, 128)
        case.update(causal=rng.random() < 0.8, seqs=seqs, tokens=max(seqs, _log_int(rng, 16, 32768)),
                    mix=rng.randrange(1 << 20), spare=rng.choice((0, 0, 0, 7, 300)), padded=rng.random() < 0.25)
        if case["padded"]:
            case["tokens"] -= case["tokens"] % seqs
        if work(case)["flops"] * _cost(case) <= limit:
            return case


def _cost(case):
    """float32 products run at a sixteenth of the 16-bit rate at most."""
    return 16 if case["dtype"] == "fp32" else 1


# -- what a program has in hand ---------------------------------------------

def _lengths(case):
    """Each sequence's tokens: those of a server's queue, a few long among many short, one in nine empty."""
    rng = random.Random(case["mix"])
    n, total = case["seqs"], case["tokens"]
    if case["padded"]:  # right-padded to the longest
        each = total // n
        return [each if b == 0 else rng.randint(each // 4, each) for b in range(n)]
    share = [0.0 if b % 9 == 8 else 0.2 + rng.expovariate(1.0) for b in range(n)]
    whole = sum(share)
    lengths = [int(total * x / whole) for x in share]
    lengths[0] += total - sum(lengths)
    return lengths


def _cache_lengths(case):
    """From the whole capacity down to a quarter; room for the drafted tokens at the least."""
    b, longest = case["batch"], case["capacity"]
    return [max(case["new"], longest - (longest - longest // 4) * i // b) for i in range(b)]


def _tree(case, rng):
    """Parents of a batch's drafted tokens. Every third sequence has fewer drafts: its last slots are empty."""
    parents = []
    for b in range(case["batch"]):
        t = case["new"]
        used = t if b % 3 else max(1, t - t // 4)
        row = [-1 if i == 0 or rng.random() < 0.1 else rng.randint(max(0, i - 8), i - 1) for i in range(used)]
        parents.append(row + [t] * (t - used))
    return parents


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, h, hk, d, dv = (DTYPES[case["dtype"]], *(case[n] for n in ("heads", "kv_heads", "dim", "dim_v")))

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0, std, generator=g)

    state = {"case": case}
    if case["kind"] == "tree":
        b, t, cap = case["batch"], case["new"], case["capacity"]
        state["q"] = normal(b, t, h, d, std=1.5).transpose(1, 2)  # as a projection gives it
        state["k"], state["v"] = normal(b, hk, cap, d), normal(b, hk, cap, dv)
        lengths = _cache_lengths(case)
        rng.shuffle(lengths)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
        state["host_lengths"] = lengths
        state["parents"] = torch.tensor(_tree(case, rng), dtype=torch.int32).cuda() if case["tree"] else None
        return state
    lengths = _lengths(case)
    rng.shuffle(lengths)
    room = [case["tokens"] // case["seqs"]] * case["seqs"] if case["padded"] else lengths
    starts = [0]
    for n in room:
        starts.append(starts[-1] + n)
    rows = case["tokens"] + case["spare"]
    state["offsets"] = torch.tensor(starts, dtype=torch.int32).cuda()
    state["valid_len"] = torch.tensor(lengths, dtype=torch.int32).cuda() if case["padded"] else None
    state["spans"] = [(s, n) for s, n in zip(starts, lengths) if n > 0]
    # One projection's output, split into heads as views.
    fused = normal(rows, h * d + hk * (d + dv))
    q, k, v = fused.split((h * d, hk * d, hk * dv), 1)
    q.mul_(1.5)
    state["q"], state["k"], state["v"] = q.view(rows, h, d), k.view(rows, hk, d), v.view(rows, hk, dv)
    if case["kind"] == "train":
        state["dout"] = normal(rows, h, dv, std=0.1)
        for name in ("q", "k", "v"):
            state[name] = state[name].detach().requires_grad_()
    return state


# -- one pass -----------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_tree(state) if state["case"]["kind"] == "tree" else _plain_packed(state)


def _run_own(state):
    from techjam_amd.kernels import packed_attention, tree_attention

    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    if case["kind"] == "tree":
        with torch.no_grad():
            return tree_attention(q, k, v, state["lengths"], state["parents"])
    if case["kind"] == "attend":
        with torch.no_grad():
            return packed_attention(q, k, v, state["offsets"], is_causal=case["causal"], valid_len=state["valid_len"])
    out = packed_attention(q, k, v, state["offsets"], is_causal=case["causal"], valid_len=state["valid_len"])
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"])]


def _plain_softmax(scores, seen):
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.max(-1, keepdim=True).values
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_packed(state):
    """One sequence at a time, its heads together, as many rows at once as give 2^28 scores."""
    case = state["case"]
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    rows, h, d = q.shape
    hk, dv = k.shape[1], v.shape[-1]
    g, scale, train = h // hk, d ** -0.5, case["kind"] == "train"
    out = torch.zeros(rows, h, dv, dtype=q.dtype, device=q.device)
    if train:
        grads = [torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
    for start, n in state["spans"]:
        span = slice(start, start + n)
        # [key head, group, token, dim]
        qs = q[span].float().view(n, hk, g, d).permute(1, 2, 0, 3)
        ks = k[span].float().permute(1, 0, 2)[:, None]
        vs = v[span].float().permute(1, 0, 2)[:, None]
        step = max(64, (1 << 28) // (h * n))
        if train:
            dk, dvv = torch.zeros(hk, n, d, device=q.device), torch.zeros(hk, n, dv, device=q.device)
        for first in range(0, n, step):
            last = min(n, first + step)
            keys = last if case["causal"] else n
            i = torch.arange(first, last, device=q.device)
            j = torch.arange(keys, device=q.device)
            seen = j[None, :] <= i[:, None] if case["causal"] else torch.ones(last - first, keys, dtype=torch.bool,
                                                                              device=q.device)
            qb, kb, vb = qs[:, :, first:last], ks[:, :, :keys], vs[:, :, :keys]
            p = _plain_softmax(torch.matmul(qb, kb.transpose(-1, -2)) * scale, seen)
            at = slice(start + first, start + last)
            out[at] = torch.matmul(p, vb).permute(2, 0, 1, 3).reshape(last - first, h, dv).to(out.dtype)
            if not train:
                continue
            do = state["dout"][at].float().view(last - first, hk, g, dv).permute(1, 2, 0, 3)
            dvv[:, :keys] += torch.matmul(p.transpose(-1, -2), do).sum(1)
            dp = torch.matmul(do, vb.transpose(-1, -2))
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            del p, dp
            grads[0][at] = torch.matmul(ds, kb).permute(2, 0, 1, 3).reshape(last - first, h, d).to(q.dtype)
            dk[:, :keys] += torch.matmul(ds.transpose(-1, -2), qb).sum(1)
        if train:
            grads[1][span] = dk.transpose(0, 1).to(k.dtype)
            grads[2][span] = dvv.transpose(0, 1).to(v.dtype)
    return [out, *grads] if train else out


def _plain_lineage(state):
    """Truth values [sequence, token, token]: which drafted tokens each one sees. Empty slots see none."""
    case, parents = state["case"], state["parents"]
    t = case["new"]
    i = torch.arange(t, device=state["q"].device)
    if parents is None:
        return (i[None, :] <= i[:, None]).expand(case["batch"], t, t)
    used = (parents >= -1) & (parents < i)
    step = ((parents[:, :, None] == i) & used[:, :, None]).float() + torch.eye(t, device=i.device)
    reach = step
    for _ in range(max(1, t - 1).bit_length()):  # lineages of twice the length
        reach = (torch.matmul(reach, reach) > 0).float()
    return (reach > 0) & used[:, :, None]


def _plain_tree(state):
    """One sequence at a time, its heads together, over its own keys."""
    q, k, v = state["q"], state["k"], state["v"]
    b_all, h, t, d = q.shape
    hk, dv = k.shape[1], v.shape[-1]
    g = h // hk
    lineage = _plain_lineage(state)
    out = torch.empty(b_all, h, t, dv, dtype=q.dtype, device=q.device)
    for b, n in enumerate(state["host_lengths"]):
        seen = torch.ones(t, n, dtype=torch.bool, device=q.device)
        seen[:, n - t:] = lineage[b]
        seen &= lineage[b].any(-1, keepdim=True)
        qb = q[b].float().reshape(hk, g * t, d)
        scores = torch.matmul(qb, k[b, :, :n].float().transpose(-1, -2)) * d ** -0.5
        p = _plain_softmax(scores.view(hk, g, t, n), seen).view(hk, g * t, n)
        out[b] = torch.matmul(p, v[b, :, :n].float()).view(h, t, dv).to(out.dtype)
    return out


# -- what a pass cannot do without --------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    h, hk, d, dv = (case[n] for n in ("heads", "kv_heads", "dim", "dim_v"))
    if case["kind"] == "tree":
        # Each drafted token sees the keys before the drafts and, at the least, itself.
        lengths, t = _cache_lengths(case), case["new"]
        pairs = sum(t * (n - t) + t for n in lengths)
        moved = sum(lengths) * hk * (d + dv) + len(lengths) * t * h * (d + dv)
        return {"bytes": float(size * moved), "flops": float(pairs * h * 2 * (d + dv))}
    lengths = _lengths(case)
    tokens, rows = sum(lengths), case["tokens"] + case["spare"]
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
    moved = tokens * (h * d + hk * (d + dv)) + rows * h * dv
    flops = pairs * h * 2 * (d + dv)
    if case["kind"] == "train":
        # The scores' gradient, and q's, k's and v's: four more products a pair.
        moved += tokens * h * dv + rows * (h * d + hk * (d + dv))
        flops += pairs * h * 4 * (d + dv)
    return {"bytes": float(size * moved), "flops": float(flops)}


# -- the definition in 64 bits --------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return _exact_tree(state) if case["kind"] == "tree" else _exact_packed(state)


def _exact_rows(q, k, v, first):
    """softmax(q k^T / sqrt d) v of rows whose first sees the keys up to ``first`` (None: every row sees all)."""
    scores = q @ k.mT / math.sqrt(q.shape[-1])
    if first is not None:
        later = torch.ones(scores.shape, dtype=torch.bool, device=q.device).triu(first + 1)
        scores.masked_fill_(later, -math.inf)
    return torch.softmax(scores, -1) @ v


def _exact_packed(state):
    """One head of one sequence at a time, 2048 rows at once, with torch's own gradients."""
    case = state["case"]
    train = case["kind"] == "train"
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    g = q.shape[1] // k.shape[1]
    f64 = dict(dtype=torch.float64, device=q.device)
    out = torch.zeros(*q.shape[:2], v.shape[-1], **f64)
    grads = [torch.zeros(t.shape, **f64) for t in (q, k, v)]
    for start, n in state["spans"]:
        for head in range(q.shape[1]):
            kv = head // g
            for r0 in range(0, n, 2048):
                r1 = min(n, r0 + 2048)
                end = start + (r1 if case["causal"] else n)
                leaves = [q[start + r0:start + r1, head].double(), k[start:end, kv].double(), v[start:end, kv].double()]
                if train:
                    leaves = [t.requires_grad_() for t in leaves]
                o = _exact_rows(*leaves, r0 if case["causal"] else None)
                out[start + r0:start + r1, head] = o.detach()
                if train:
                    dout = state["dout"][start + r0:start + r1, head].double()
                    dq, dk, dvv = torch.autograd.grad(o, leaves, dout)
                    grads[0][start + r0:start + r1, head] += dq
                    grads[1][start:end, kv] += dk
                    grads[2][start:end, kv] += dvv
    return [out, *grads] if train else out


def _exact_tree(state):
    """Each drafted token's own lineage, followed from parent to parent, and one head at a time over those keys."""
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    b_all, h, t, _ = q.shape
    g = h // k.shape[1]
    parents = state["parents"].tolist() if case["tree"] else [[i - 1 for i in range(t)]] * b_all
    out = torch.zeros(b_all, h, t, v.shape[-1], dtype=torch.float64, device=q.device)
    for b, n in enumerate(state["host_lengths"]):
        hidden = torch.zeros(t, n, dtype=torch.bool)
        live = []
        for i in range(t):
            hidden[i, n - t:] = True
            at = i
            while -1 <= parents[b][at] < at:
                hidden[i, n - t + at] = False
                if parents[b][at] == -1:
                    live.append(i)
                    break
                at = parents[b][at]
        hidden = hidden.to(q.device)[live]
        for kv in range(k.shape[1]):
            keys, values = k[b, kv, :n].double(), v[b, kv, :n].double()
            for head in range(kv * g, kv * g + g):
                scores = q[b, head, live].double() @ keys.mT / math.sqrt(q.shape[-1])
                out[b, head, live] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ values
    return out
