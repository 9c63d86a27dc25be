"""Operators over trees of drafted tokens, as a step of speculative decoding uses them: what is measured, in plain torch and through
``vllm_cpp_b200.ops.draft_tree``.

A step holds for each request ``n`` nodes (rows ``starts[r]..starts[r + 1]``): node 0 is the last accepted token, the others are
drafts, each with an earlier node as its parent. Node ``j`` has its keys and values in the cache at position ``c + j`` behind the
``c`` tokens of the request's context.

``mask``: for every node the bits of its ancestors and itself (64 nodes a word), and its position, ``c`` plus its depth.
``attention``: a node sees its context and the nodes of its bits.
``verify``: from the root down, each child is accepted or refused by a given random number so that the tokens that come out have
the target's distribution; where no child is accepted the last token is drawn from what remains of it.
``compact``: the cells of the accepted nodes move together behind the context, in every layer.
"""
import math
import random

import torch

own = False

MASK64 = (1 << 64) - 1


def listed():
    m = dict(op="mask", most=64)
    a = dict(op="attention", page=32, d=128, hq=32, hkv=8, window=0, softcap=0.0, empty=False)
    v = dict(op="verify", temperature=1.0, keep=0)
    k = dict(op="compact", page=32, d=128)
    cases = {
        # one user's tree of a step
        "mask, one tree": dict(m, reqs=1, n_low=60, n_high=60, wide=4),
        # a full server's trees, some larger than a word
        "mask, 256 trees": dict(m, most=128, reqs=256, n_low=9, n_high=101, wide=5),
        # one user in a chat, a small tree
        "attention, one chat": dict(a, reqs=1, n_low=16, n_high=16, c_low=1000, c_high=1000),
        # one user with a long document, a large tree
        "attention, one long context": dict(a, reqs=1, n_low=61, n_high=61, c_low=120000, c_high=120000),
        # a loaded server, ragged contexts and trees, eight query heads a key head
        "attention, 48 requests": dict(a, hkv=4, reqs=48, n_low=5, n_high=26, c_low=100, c_high=4000),
        # a full server
        "attention, 128 requests": dict(a, reqs=128, n_low=32, n_high=32, c_low=200, c_high=3800),
        # 64-dim heads in a sliding window with capped scores
        "attention, window": dict(a, d=64, hq=24, reqs=33, n_low=1, n_high=37, c_low=1, c_high=9000, window=1024, softcap=30.0),
        # one user's chain from a draft model
        "verify, one chain": dict(v, reqs=1, n_low=5, n_high=5, wide=1, vocab=128256, drawn=True),
        # a server's chains of one to five drafts from a draft model
        "verify, 64 chains": dict(v, reqs=64, n_low=2, n_high=6, wide=1, vocab=151936, drawn=True),
        # trees of a draft head's likeliest tokens
        "verify, 24 trees": dict(v, reqs=24, n_low=31, n_high=48, wide=4, vocab=128256, drawn=False),
        # one user's accepted path in 32 layers
        "compact, one path": dict(k, reqs=1, layers=32, hkv=8, nodes=60, steps_low=4, steps_high=4, c_high=700),
        # a server's accepted paths of up to seven drafts
        "compact, 64 paths": dict(k, reqs=64, layers=16, hkv=8, nodes=40, steps_low=0, steps_high=7, c_high=60),
    }
    return [dict(name=k, **v) for k, v in cases.items()]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["mask", "attention", "attention", "attention", "verify", "verify", "compact"])
    if op == "mask":
        most = rng.choice([64, 64, 128, 256])
        high = log(1, most)
        return dict(op=op, most=most, reqs=log(1, 300), n_low=log(1, high), n_high=high, wide=rng.randint(1, 6))
    if op == "compact":
        steps = rng.randint(1, 9)
        return dict(op=op, page=rng.choice([16, 32, 64]), d=rng.choice([64, 128, 256]), reqs=log(1, 40), layers=log(2, 16), hkv=rng.choice([1, 2, 4, 8]),
                    nodes=rng.randint(2 * steps + 2, 64), steps_low=rng.randint(0, steps), steps_high=steps, c_high=log(1, 150))
    if op == "verify":
        vocab = rng.choice([log(300, 30000), 32000, 50257, 128256, 151936, 152063])
        wide = rng.choice([1, 1, 2, 4])
        reqs = log(1, 64)
        high = log(1, max(2, min(48, 9_000_000 // (reqs * vocab // 16))))
        return dict(op=op, reqs=reqs, n_low=log(1, high), n_high=high, wide=wide, vocab=vocab, drawn=rng.random() < 0.6,
                    temperature=rng.choice([1.0, 1.0, 0.0, 0.5]), keep=rng.choice([0, 0, 0, 50]))
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    while hkv * group > 32:
        group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    reqs = log(1, 64)
    n_high = log(1, max(2, min(130, 3000 // reqs)))
    c_high = min(60000, log(1, max(2, 120000 // reqs)))
    return dict(op=op, page=rng.choice([16, 32, 64, 128]), d=rng.choice([64, 128, 128, 256]), hq=hkv * group, hkv=hkv,
                window=rng.choice([0, 0, 0, log(16, 4000)]), softcap=rng.choice([0.0, 0.0, 0.0, 25.0]), empty=rng.random() < 0.2, reqs=reqs,
                n_low=log(1, n_high), n_high=n_high, c_low=rng.choice([0, rng.randint(0, c_high)]), c_high=c_high)


# ------------------------------------------------------------------------------------------------ inputs
def _spread(n, low, high):
    """``n`` lengths between ``low`` and ``high`` in an order that jumps about."""
    return [low + (high - low) * ((i * 7919 + n * 31) % 97) // 96 for i in range(n)]


def _sizes(c):
    """Nodes of each request, tokens of its context."""
    return _spread(c["reqs"], c["n_low"], c["n_high"]), _spread(c["reqs"], c.get("c_low", 0), c.get("c_high", 500))[::-1]


def _trees(sizes, wide, rng):
    """Parents of all nodes, within their request: chains for ``wide`` 1, else trees of at most ``wide`` children a node and eight
    nodes below the root one under another."""
    parents = []
    for n in sizes:
        level, count = [0], [0] * n
        parents.append(-1)
        for j in range(1, n):
            free = [i for i in range(j) if count[i] < wide and level[i] < 8] if wide > 1 else [j - 1]
            p = min(rng.choice(free), rng.choice(free))
            count[p] += 1
            level.append(level[p] + 1)
            parents.append(p)
    return parents


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(sizes):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return _ints(at)


def _page_table(lengths, page, gen):
    """Pages of the requests, in no order; page 0 belongs to none. Behind a request's pages: page 0."""
    counts = [max(1, -(-n // page)) for n in lengths]
    total = sum(counts) + 1
    perm = (torch.randperm(total - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    table = torch.zeros((len(lengths), max(counts)), dtype=torch.int32, device="cuda")
    table[torch.arange(max(counts), device="cuda")[None] < _ints(counts)[:, None]] = perm
    return table, total


def _normal_bf16(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def _peaked(rows, vocab, gen):
    """Logits with a few likely tokens a row, as a language model has them."""
    x = torch.randn((rows, vocab), generator=gen, device="cuda")
    at = torch.randint(0, vocab, (rows, 8), generator=gen, device="cuda")
    return x.scatter_add_(1, at, 4 + 12 * torch.rand((rows, 8), generator=gen, device="cuda"))


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": c}
    if c["op"] == "compact":
        contexts = _spread(c["reqs"], 0, c["c_high"])
        lengths = [n + c["nodes"] for n in contexts]
        s["table"], pages = _page_table(lengths, c["page"], gen)
        s["caches"] = _normal_bf16((c["layers"], pages, 2, c["page"], c["hkv"], c["d"]), gen)
        s["layers"] = list(s["caches"])
        s["lengths"], s["starts"] = _ints(lengths), _starts([c["nodes"]] * c["reqs"])
        steps = _spread(c["reqs"], c["steps_low"], c["steps_high"])
        path = torch.full((c["reqs"], c["steps_high"] + 1), -1, dtype=torch.int32)
        for r, k in enumerate(steps):                    # the accepted nodes lie behind the places that they move to
            path[r, 0] = 0
            path[r, 1: k + 1] = torch.tensor(sorted(rng.sample(range(c["steps_high"] + 1, c["nodes"]), k)), dtype=torch.int32)
        s["path"] = path.cuda()
        return s
    sizes, contexts = _sizes(c)
    rows = sum(sizes)
    s["starts"] = _starts(sizes)
    s["most_n"] = max(sizes)
    parents = _trees(sizes, c.get("wide", 4), rng)
    s["parents"] = _ints(parents)
    if c["op"] == "verify":
        vocab = c["vocab"]
        s["logits"] = _peaked(rows, vocab, gen)
        guess = s["logits"] + 0.7 * torch.randn((rows, vocab), generator=gen, device="cuda")
        if c["keep"]:                                    # what a top-k filter leaves of them
            least = s["logits"].topk(min(c["keep"], vocab), 1).values[:, -1:]
            s["logits"] = torch.where(s["logits"] < least, -math.inf, s["logits"])
        parent_row = torch.repeat_interleave(s["starts"][:-1].long(), s["starts"].diff().long()) + s["parents"].long().clamp(min=0)
        if c["drawn"]:
            s["probs"] = torch.softmax(guess, 1)
            s["tokens"] = torch.multinomial(s["probs"][parent_row], 1, generator=gen)[:, 0]
        else:
            seen, rank = {}, []
            for i, p in enumerate(parent_row.tolist()):
                rank.append(seen.get(p, 0))
                seen[p] = rank[-1] + 1
            best = guess.topk(max(rank) + 1, 1).indices
            s["probs"], s["tokens"] = None, best[parent_row, _ints(rank, torch.int64)]
        s["chain"] = c["wide"] == 1
        s["most_children"] = c["wide"]
        s["uniforms"] = torch.rand(rows, generator=gen, device="cuda")
        s["seeds"] = torch.randint(-2 ** 62, 2 ** 62, (c["reqs"],), generator=gen, device="cuda")
        s["steps"] = torch.randint(0, 5000, (c["reqs"],), generator=gen, device="cuda")
        warm = torch.rand(c["reqs"], generator=gen, device="cuda") < c["temperature"]
        s["temperature"] = torch.where(warm, 0.8, 0.0)   # (greedy requests stand among sampled ones)
        s["most_tokens"] = c["n_high"] if c["wide"] == 1 else min(c["n_high"], 9)
        return s
    lengths = [a + b for a, b in zip(sizes, contexts)]
    s["lengths"] = _ints(lengths)
    if c["op"] == "mask":
        return s
    s["bits"], s["positions"] = _mask_plain(s, max(1, -(-max(sizes) // 64)))
    if c["empty"]:                                       # rows of padding nodes see nothing of the tree
        s["bits"][torch.rand(rows, generator=gen, device="cuda") < 0.2] = 0
    s["table"], pages = _page_table(lengths, c["page"], gen)
    s["cache"] = _normal_bf16((pages, 2, c["page"], c["hkv"], c["d"]), gen)
    merged = _normal_bf16((rows, (c["hq"] + 2 * c["hkv"]) * c["d"]), gen).mul_(3)      # scores of a spread of about three
    s["q"] = merged[:, : c["hq"] * c["d"]]               # as the projection of q, k and v leaves them
    s["out"] = torch.empty((rows, c["hq"] * c["d"]), dtype=torch.bfloat16, device="cuda")
    s["most_length"] = max(lengths)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _of_rows(starts, rows):
    """(request, node) of each row."""
    r = torch.repeat_interleave(torch.arange(starts.numel() - 1, device="cuda"), starts.diff().long(), output_size=rows)
    return r, torch.arange(rows, device="cuda") - starts[r]


def _above(s):
    """[requests, n, n] truth values: node j is node i or above it."""
    rows, most = s["parents"].numel(), s["most_n"]
    r, j = _of_rows(s["starts"], rows)
    up = torch.zeros((s["starts"].numel() - 1, most, most), device="cuda")
    up[r, j, j] = 1
    up[r, j, torch.where(s["parents"] < 0, j, s["parents"].long())] = 1
    for _ in range(max(1, (most - 1).bit_length())):     # all walks of 2, 4, 8.. steps
        up = (up @ up > 0).float()
    return up > 0


def _mask_plain(s, words):
    r, j = _of_rows(s["starts"], s["parents"].numel())
    above = _above(s)[r, j]                              # [rows, n]
    bits = torch.nn.functional.pad(above.long(), (0, 64 * words - above.shape[1])).view(-1, words, 64)
    bits = (bits << torch.arange(64, device="cuda")).sum(-1)
    context = s["lengths"].long() - s["starts"].diff()
    return bits, context[r] + above.sum(-1) - 1


def _attention_plain(s):
    c = s["case"]
    d, hq, hkv, page = c["d"], c["hq"], c["hkv"], c["page"]
    rows, most, keys = s["q"].shape[0], s["most_n"], s["most_length"]
    r, j = _of_rows(s["starts"], rows)
    kv = s["cache"][s["table"].long()]                   # [requests, pages, 2, page, hkv, d]
    k, v = (kv[:, :, i].flatten(1, 2)[:, :keys].permute(0, 2, 3, 1).float() for i in (0, 1))
    q = torch.zeros((c["reqs"], most, hq, d), device="cuda")
    q[r, j] = s["q"].view(rows, hq, d).float()
    z = q.view(c["reqs"], most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).flatten(2, 3) @ k / math.sqrt(d)
    if c["softcap"] > 0:
        z = c["softcap"] * torch.tanh(z / c["softcap"])
    at = torch.arange(keys, device="cuda")
    context = (s["lengths"] - s["starts"].diff())[r].long()[:, None]
    node = at - context                                  # [rows, keys]
    inside = (node >= 0) & (at < s["lengths"][r][:, None])
    word = s["bits"].gather(1, (node // 64).clamp(0, s["bits"].shape[1] - 1))
    seen = torch.where(node < 0, torch.ones_like(node, dtype=torch.bool), inside & ((word >> (node % 64)) & 1 > 0))
    if c["window"] > 0:
        seen &= (node >= 0) | (at > s["positions"][:, None] - c["window"])
    all_seen = torch.zeros((c["reqs"], most, keys), dtype=torch.bool, device="cuda")
    all_seen[r, j] = seen
    z = z.view(c["reqs"], hq, most, keys).masked_fill_(~all_seen[:, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = p.view(c["reqs"], hkv, -1, keys) @ v.transpose(2, 3)
    o = o.view(c["reqs"], hq, most, d) / torch.where(total == 0, torch.ones_like(total), total)
    return o.transpose(1, 2)[r, j].flatten(1).to(torch.bfloat16)


def _shifted(z, n):
    """``z`` as an unsigned number, shifted right."""
    return (z >> n) & ((1 << (64 - n)) - 1)


def _signed(z):
    return z - (1 << 64) if z >> 63 else z


def _split_mix(z):
    z = z + _signed(0x9E3779B97F4A7C15)
    z = (z ^ _shifted(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shifted(z, 27)) * _signed(0x94D049BB133111EB)
    return z ^ _shifted(z, 31)


def _exponentials(seeds, steps, vocab):
    """[requests, vocab] exponentially distributed numbers that seeds and steps name."""
    col = torch.arange(vocab, device="cuda")
    z = _split_mix(seeds[:, None] ^ _split_mix(steps[:, None] * 0x100000001B3 + col))
    return -torch.log((_shifted(z, 11).double() + 0.5) / 2.0 ** 53)


def _verify_plain(s):
    """In 64 bits, as a random number may lie next to the border that it is compared with."""
    logits, probs, tokens = s["logits"], s["probs"], s["tokens"]
    rows, vocab = logits.shape
    r, j = _of_rows(s["starts"], rows)
    root, first = j == 0, s["starts"][:-1].long()
    parent = torch.where(root, torch.arange(rows, device="cuda"), first[r] + s["parents"].clamp(min=0))
    # which of its parent's children a node is: as many as come before it
    before = (parent[:, None] == parent[None]) & ~root[:, None] & ~root[None]
    rank = (before & (torch.arange(rows, device="cuda")[None] < torch.arange(rows, device="cuda")[:, None])).sum(1)
    w = torch.exp(logits.double() - logits.amax(1, keepdim=True))
    best = logits.argmax(1)
    greedy = (s["temperature"] < 1e-5)[r]
    z, b = w.sum(1), torch.zeros(rows, dtype=torch.float64, device="cuda")
    next_ = torch.full((rows + 1,), -1, device="cuda")   # the accepted child of each row (the last place is nobody's)
    own_w = w[parent, tokens]                            # weight of a node's token where its parent chooses
    q = probs[parent, tokens].double() if probs is not None else None
    for k in range(s["most_children"]):
        now = (rank == k) & ~root
        asked = now & (next_[parent] < 0)
        if probs is not None:
            left = (own_w - b[parent] * q).clamp(min=0)
            ok = s["uniforms"].double() * q * z[parent] < left
        else:
            ok = s["uniforms"].double() * z[parent] < w[parent, tokens]
        ok = asked & torch.where(greedy, tokens == best[parent], ok)
        at = torch.arange(rows, device="cuda")
        next_.scatter_(0, torch.where(ok, parent, rows), torch.where(ok, at, -1))
        next_[rows] = -1
        no = torch.zeros(rows + 1, dtype=torch.bool, device="cuda")
        no[torch.where(asked & ~ok & ~greedy, parent, rows)] = True
        no = no[:rows]
        if probs is not None:
            b = torch.where(no, b + z, b)
            z = (w - b[:, None] * probs).clamp_(min=0).sum(1)
        else:
            gone = torch.where(asked & ~ok & ~greedy, parent, rows)
            w = torch.cat([w, w.new_zeros((1, vocab))])
            w[gone, tokens] = 0
            w = w[:rows]
            z = w.sum(1)
    # a node is on the path if every node from it to the root is its parent's choice
    chosen = root | (next_[parent] == torch.arange(rows, device="cuda"))
    wrong = torch.zeros((s["starts"].numel() - 1, s["most_n"]), device="cuda")
    wrong[r, j] = (~chosen).float()
    above = _above(s)
    on = (above.float() @ wrong[..., None])[r, j, 0] == 0
    depth = above.sum(-1)[r, j] - 1
    count = torch.zeros(s["starts"].numel() - 1, dtype=torch.int64, device="cuda").index_add_(0, r, on.long())
    path = torch.full((s["starts"].numel() - 1, s["most_tokens"] + 1), -1, dtype=torch.int32, device="cuda")
    out = torch.full_like(path, -1, dtype=torch.int64)
    place = torch.where(on, depth, s["most_tokens"])
    path[r, place] = torch.where(on, j, -1).int()
    out[r, torch.where(on & ~root, depth - 1, s["most_tokens"])] = torch.where(on & ~root, tokens, -1)
    # the last token: drawn from what remains at the path's end
    end = first + path.gather(1, (count - 1)[:, None])[:, 0]
    left = w[end]
    if probs is not None:
        left = (left - b[end, None] * probs[end]).clamp(min=0)
    last = (left / _exponentials(s["seeds"], s["steps"], vocab)).argmax(1)
    last = torch.where(s["temperature"] < 1e-5, best[end], last)
    out.scatter_(1, (count - 1)[:, None], last[:, None])
    return out[:, :-1].contiguous(), path[:, :-1].contiguous(), count.int()


def _compact_plain(s):
    c = s["case"]
    context = (s["lengths"] - s["starts"].diff()).long()[:, None]
    step = torch.arange(s["path"].shape[1], device="cuda")[None]
    there = (s["path"] >= 0) & (step > 0)

    def cell(position):
        position = torch.where(there, position, torch.zeros_like(position))
        return s["table"].long().gather(1, position // c["page"]), position % c["page"]

    (page, at), (to_page, to_at) = cell(context + s["path"].clamp(min=0)), cell(context + step)
    held = s["caches"][:, page, :, at]                   # [requests, steps, layers, 2, hkv, d], read before any is written
    s["caches"][:, to_page[there], :, to_at[there]] = held[there]
    return s["caches"]


# ----------------------------------------------------------------------------------------- the framework's operators
def _own(s):
    from vllm_cpp_b200.ops import draft_tree
    c = s["case"]
    if c["op"] == "mask":
        return draft_tree.mask(s["parents"], q_start=s["starts"], seq_lens=s["lengths"], max_nodes=c["most"])
    if c["op"] == "attention":
        return draft_tree.attention(s["q"], s["cache"], block_table=s["table"], seq_lens=s["lengths"], q_start=s["starts"], mask=s["bits"],
                                    positions=s["positions"], scale=1 / math.sqrt(c["d"]), out=s["out"], softcap=c["softcap"],
                                    window=c["window"])
    if c["op"] == "verify":
        return draft_tree.verify(s["logits"], s["tokens"], q_start=s["starts"], parents=None if s["chain"] else s["parents"],
                                 draft_probs=s["probs"], uniforms=s["uniforms"], seeds=s["seeds"], steps=s["steps"],
                                 temperature=s["temperature"], max_tokens=s["most_tokens"])
    draft_tree.compact(s["layers"], block_table=s["table"], seq_lens=s["lengths"], q_start=s["starts"], path=s["path"])
    return s["caches"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "mask":
        return _mask_plain(state, -(-state["case"]["most"] // 64))
    return _attention_plain(state) if op == "attention" else _verify_plain(state) if op == "verify" else _compact_plain(state)


def work(case):
    c = case
    if c["op"] == "compact":
        cells = sum(_spread(c["reqs"], c["steps_low"], c["steps_high"]))
        moved = cells * c["layers"] * 2 * c["hkv"] * c["d"] * 2
        return {"bytes": 2 * moved + c["reqs"] * (c["steps_high"] + 1) * 4 + cells * 8, "flops": 0}
    sizes, contexts = _sizes(c)
    rows = sum(sizes)
    if c["op"] == "mask":
        return {"bytes": 4 * rows + 8 * c["reqs"] + rows * 8 * (-(-c["most"] // 64) + 1), "flops": 0}
    if c["op"] == "verify":
        # The rows of the root and of one draft are read at the least where there are drafts; the children's tokens, and a draw.
        visited = sum(min(n, 2) for n in sizes)
        return {"bytes": visited * c["vocab"] * (8 if c["drawn"] else 4) + rows * 24, "flops": visited * c["vocab"] * (5 if c["drawn"] else 3)}
    d, hq, hkv, w = c["d"], c["hq"], c["hkv"], c["window"]
    # (a node of a tree sees its context and about half a chain of the tree's square root of nodes)
    pairs = sum(n * ((min(w, m) if w > 0 else m) + math.isqrt(n)) for n, m in zip(sizes, contexts))
    keys = sum((min(w, m) if w > 0 else m) + n for n, m in zip(sizes, contexts))
    table = sum(-(-(n + m) // c["page"]) for n, m in zip(sizes, contexts)) * 4
    return {"bytes": keys * hkv * d * 4 + 2 * rows * hq * d * 2 + table + rows * 8, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def _trees_of(s):
    """For each request: its first row and the list of its nodes' parents."""
    starts, parents = s["starts"].tolist(), s["parents"].tolist()
    return [(a, parents[a:b]) for a, b in zip(starts, starts[1:])]


def _attention_exact(s):
    c = s["case"]
    d, page, hq, hkv = c["d"], c["page"], c["hq"], c["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    bits = [[w & MASK64 for w in row] for row in s["bits"].tolist()]
    positions = s["positions"].tolist()
    for r, (first, parents) in enumerate(_trees_of(s)):
        n, total = len(parents), int(s["lengths"][r])
        context = total - n
        kv = s["cache"][s["table"][r, : -(-total // page)].long()]
        hidden = torch.zeros((n, total), dtype=torch.bool)
        for i in range(n):
            hidden[i, context:] = torch.tensor([not (bits[first + i][j // 64] >> (j % 64)) & 1 for j in range(n)])
            if c["window"] > 0:
                hidden[i, : max(0, min(context, positions[first + i] - c["window"] + 1))] = True
        hidden = hidden.cuda()
        for h in range(hkv):
            k, v = (kv[:, i, :, h].reshape(-1, d)[:total].double() for i in (0, 1))
            cols = slice(h * (hq // hkv) * d, (h + 1) * (hq // hkv) * d)
            z = torch.einsum("ngd,kd->ngk", s["q"][first: first + n, cols].double().reshape(n, hq // hkv, d), k) / math.sqrt(d)
            if c["softcap"] > 0:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            p = torch.softmax(z.masked_fill(hidden[:, None], -math.inf), -1)
            p[hidden.all(1)] = 0                          # (a row that sees nothing)
            out[first: first + n, cols] = (p @ v).reshape(n, -1)
    return out


def _numbers_exact(seed, step, vocab):
    """U of every token, by Python's whole numbers on numpy's 64-bit words."""
    import numpy as np

    def mix(z):
        z = z + np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return z ^ (z >> np.uint64(31))

    col = np.uint64((step * 0x100000001B3) & MASK64) + np.arange(vocab, dtype=np.uint64)
    z = mix(np.uint64(seed & MASK64) ^ mix(col))
    return ((z >> np.uint64(11)).astype(np.float64) + 0.5) / 9007199254740992.0


def _verify_exact(s):
    vocab, most = s["logits"].shape[1], s["most_tokens"]
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    temperature = s["temperature"].tolist()
    out, paths, counts = [], [], []
    for r, (first, parents) in enumerate(_trees_of(s)):
        at, path, said = 0, [0], []
        while True:
            row = s["logits"][first + at].double()
            children = [j for j in range(1, len(parents)) if parents[j] == at]
            taken = None
            if temperature[r] < 1e-5:
                best = int(row.argmax())
                taken = next((j for j in children if tokens[first + j] == best), None)
            else:
                p = torch.softmax(row, 0)
                q = s["probs"][first + at].double() if s["probs"] is not None else None
                for j in children:
                    x = tokens[first + j]
                    if q is not None:
                        if u[first + j] * float(q[x]) < float(p[x]):
                            taken = j
                            break
                        p = (p - q).clamp(min=0)
                    else:
                        if u[first + j] < float(p[x]):
                            taken = j
                            break
                        p = p.clone()
                        p[x] = 0
                    p = p / p.sum()
            if taken is None:
                if temperature[r] >= 1e-5:
                    e = -torch.log(torch.from_numpy(_numbers_exact(int(s["seeds"][r]), int(s["steps"][r]), vocab)).cuda())
                    best = int((p / e).argmax())
                said.append(best)
                break
            at = taken
            path.append(at)
            said.append(tokens[first + at])
        out.append(said + [-1] * (most - len(said)))
        paths.append(path + [-1] * (most - len(path)))
        counts.append(len(path))
    return _ints(out, torch.int64), _ints(paths), _ints(counts)


def _mask_exact(s):
    words = -(-s["case"]["most"] // 64)
    bits, positions = [], []
    for r, (_, parents) in enumerate(_trees_of(s)):
        held = []
        for j, p in enumerate(parents):
            held.append((held[p] if p >= 0 else 0) | 1 << j)
            bits.append([_signed(held[-1] >> (64 * i) & MASK64) for i in range(words)])
            positions.append(int(s["lengths"][r]) - len(parents) + bin(held[-1]).count("1") - 1)
    return _ints(bits, torch.int64), _ints(positions, torch.int64)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "compact":
        before = s["caches"].clone()
        starts, table, path, lengths = s["starts"].tolist(), s["table"].tolist(), s["path"].tolist(), s["lengths"].tolist()
        for r, steps in enumerate(path):
            base = lengths[r] - (starts[r + 1] - starts[r])
            for i, node in enumerate(steps):
                if i and node >= 0:
                    a, b = base + node, base + i
                    s["caches"][:, table[r][b // case["page"]], :, b % case["page"]] = before[:, table[r][a // case["page"]], :, a % case["page"]]
        return s["caches"].double() if s["caches"].numel() < 1 << 29 else None
    return _mask_exact(s) if op == "mask" else _attention_exact(s) if op == "attention" else _verify_exact(s)


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(i)) for i in range(5)]:
        print(case.get("name", "drawn"), case, work(case))
