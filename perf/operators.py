"""Workloads of the speculative-decoding operators: the 8-bit key/value cache, attention for a tree of drafted
tokens over a cache, and the verification of drafted tokens against the target model's probabilities.

A case is a dict of plain values whose "kind" names one of the uses below; `prepare` makes what a serving
program holds before the call, `run` is one pass, `work` the bytes and operations the pass cannot do without,
`exact` the result in 64 bits.  With `own` false `run` computes the operators' definitions with elementary
torch operations, with `own` true it calls pluto_b200.layers.

    write    rows of keys and values are quantised into an 8-bit cache and read back as the values they hold
    commit   after a verification: the drafts' rows are written, the accepted path's rows move to the front
             of the drafts' slots, and the slots are read back
    attend   every drafted token of a tree attends to its sequence's cached tokens and to its own ancestors
    verify   drafted tokens are accepted or rejected with given random numbers, and one more token is drawn

The 8-bit cache holds E4M3 codes and one scale per (token, head) row: the smallest power of two 2^n, n >= -127,
with max|x| <= 448 * 2^n, stored as the byte n + 127; a row that is not finite holds 255 and reads back as NaN.
"""
import math
import random

import torch

own = False

# Head shapes the engine is used with: (query heads, key/value heads, head width).  40/8/128 is the configuration
# its prefill and decode are benchmarked on, 24/4/256 the default of FullAttentionParameters, 12/12/64 GPT-2 small,
# 5/1/128 one of eight GPUs' share of the first.
SHAPES = ((40, 8, 128), (24, 4, 256), (12, 12, 64), (5, 1, 128))
VOCABULARIES = (32000, 50257, 65537, 100003, 131071)


def listed():
    return [
        # one new token for each of 64 sequences in a paged cache: latency
        dict(name="write b64 1 token", kind="write", batch=64, tokens=1, longest=700, heads=8, dim=128, page=16, bf16=True),
        # three prompts of odd length, activations kept in fp32
        dict(name="write b3 2731 fp32", kind="write", batch=3, tokens=2731, longest=1, heads=4, dim=256, page=0, bf16=False),
        # a full batch of prompts: bandwidth
        dict(name="write b16 8191", kind="write", batch=16, tokens=8191, longest=1, heads=8, dim=128, page=64, bf16=True),
        # the cache step after a verification, one layer
        dict(name="commit b32 31 drafts", kind="commit", batch=32, nodes=31, longest=1500, heads=8, dim=128, page=16, bf16=True),
        # one user, one token over an 8-bit cache, output gate on: latency
        dict(name="attend b1 1 24/4/256 e4m3", kind="attend", batch=1, nodes=1, longest=777, q_heads=24, kv_heads=4, dim=256,
             page=0, eight=True, gate=True, tree=False),
        # a few users with small trees in a paged bf16 cache, output gate on
        dict(name="attend b4 13 24/4/256 bf16", kind="attend", batch=4, nodes=13, longest=3000, q_heads=24, kv_heads=4, dim=256,
             page=64, eight=False, gate=True, tree=True),
        # plain decoding of a serving batch over an 8-bit cache: the memory system
        dict(name="attend b24 1 40/8/128 e4m3", kind="attend", batch=24, nodes=1, longest=8192, q_heads=40, kv_heads=8, dim=128,
             page=64, eight=True, gate=False, tree=False),
        # a short chain of drafts for many small sequences
        dict(name="attend b24 8 12/12/64 bf16", kind="attend", batch=24, nodes=8, longest=1023, q_heads=12, kv_heads=12, dim=64,
             page=16, eight=False, gate=False, tree=False),
        # large trees over long contexts: the tensor cores
        dict(name="attend b16 61 40/8/128 e4m3", kind="attend", batch=16, nodes=61, longest=8191, q_heads=40, kv_heads=8, dim=128,
             page=64, eight=True, gate=False, tree=True),
        # one user, a chain of five sampled drafts
        dict(name="verify b1 chain 5", kind="verify", batch=1, nodes=5, vocab=50257, tree=False),
        # a serving batch, chains of eight sampled drafts
        dict(name="verify b64 chain 8", kind="verify", batch=64, nodes=8, vocab=131071, tree=False),
        # a serving batch, trees of the draft model's likeliest tokens
        dict(name="verify b32 tree 31", kind="verify", batch=32, nodes=31, vocab=50257, tree=True),
    ]


def _log(rng, low, high):
    """An integer whose logarithm is uniform, so that odd sizes come as often as round ones."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(("write", "commit", "attend", "attend", "attend", "verify", "verify"))
    hq, hkv, dim = rng.choice(SHAPES)
    page = rng.choice((0, 16, 64))
    if kind == "write":
        batch = _log(rng, 1, 64)
        return dict(kind=kind, batch=batch, tokens=_log(rng, 1, max(1, 25600000 // (batch * hkv * dim))), longest=_log(rng, 1, 2000),
                    heads=hkv, dim=dim, page=page, bf16=rng.random() < 0.7)
    if kind == "commit":
        return dict(kind=kind, batch=_log(rng, 1, 48), nodes=_log(rng, 2, 64), longest=_log(rng, 1, 3000), heads=hkv, dim=dim,
                    page=page, bf16=True)
    if kind == "attend":
        batch, nodes = _log(rng, 1, 24), _log(rng, 1, 64)
        return dict(kind=kind, batch=batch, nodes=nodes, longest=_log(rng, 1, 8192 if batch * nodes <= 500 else 4000), q_heads=hq, kv_heads=hkv,
                    dim=dim, page=page, eight=rng.random() < 0.5, gate=rng.random() < 0.3, tree=rng.random() < 0.6)
    batch = _log(rng, 1, 64)
    return dict(kind=kind, batch=batch, nodes=_log(rng, 1, max(2, min(63, 900 // batch))), vocab=rng.choice(VOCABULARIES), tree=rng.random() < 0.5)


def _lengths(case):
    """Cached tokens of every sequence before the call: the longest, and others spread below it."""
    rng = random.Random(case["batch"] * 65537 + case["longest"])
    return [case["longest"]] + [rng.randint(case["longest"] // 4, case["longest"]) for _ in range(case["batch"] - 1)]


def _counts(case):
    """Drafted tokens of every sequence: trees are ragged, chains of one length."""
    if not case["tree"]:
        return [case["nodes"]] * case["batch"]
    rng = random.Random(case["batch"] * 8191 + case["nodes"])
    return [case["nodes"]] + [rng.randint((case["nodes"] + 1) // 2, case["nodes"]) for _ in range(case["batch"] - 1)]


def _accepted(case):
    """Accepted tokens of every sequence in a commit."""
    rng = random.Random(case["batch"] * 131 + case["nodes"])
    return [rng.randint(0, min(8, case["nodes"])) for _ in range(case["batch"])]


def _power(n):
    """2^n in fp32 for whole n >= -127, from the bits: a power function may be an ulp off."""
    return ((n.clamp(min=-126) + 127) << 23).view(torch.float32) * torch.where(n < -126, 0.5, 1.0)


def _quantise(x):
    """E4M3 codes and the scale byte of every row of x [..., D]."""
    x = x.float()
    largest = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(largest)
    n = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-127)
    n = torch.where(largest > 0, n, torch.full_like(n, -127))
    fine = torch.isfinite(largest)
    n = torch.where(fine, n, torch.zeros_like(n))
    codes = (x * _power(-n)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(fine[..., None], codes, torch.full_like(codes, 0x7f))
    scale = torch.where(fine, n + 127, torch.full_like(n, 255)).to(torch.uint8)
    return codes, scale


def _values(codes, scale):
    """What codes and scale bytes stand for, in fp32."""
    n = scale.int()
    factor = torch.where(n == 255, math.nan, _power((n - 127).clamp(max=127)))
    return codes.view(torch.float8_e4m3fn).float() * factor[..., None]


def _rows(state, slots):
    """Rows of the flattened pool that hold the given slots [B, T] of the sequences."""
    page = state["page"]
    return state["table"].long().gather(1, slots // page) * page + slots % page


def _pool(case, capacity, dtype, fill):
    """Page pools for keys and values with the pages of every sequence scattered, or one page per sequence."""
    page = case["page"] or capacity
    blocks = -(-capacity // page)
    pages = case["batch"] * blocks
    table = torch.arange(pages, device="cuda") if not case["page"] else torch.randperm(pages, device="cuda", generator=fill)
    heads = case.get("heads", case.get("kv_heads"))
    new = lambda: torch.zeros(pages, page, heads, case["dim"], dtype=dtype, device="cuda")  # noqa: E731
    return page, table.to(torch.int32).view(case["batch"], blocks), new(), new()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    uniform = lambda *s: torch.rand(*s, device="cuda", generator=gen)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch, kind = case["batch"], case["kind"]
    if kind == "verify":
        nodes, vocab = case["nodes"], case["vocab"]
        # the draft model's logits are the target's with an error; both are peaked as a language model's are
        logits = normal(batch, nodes + 1, vocab) * 6
        if case["tree"]:
            parents = (uniform(batch, nodes) * torch.arange(1, nodes + 1, device="cuda")).int() - 1
            guess = torch.topk(logits + normal(batch, nodes + 1, vocab), 16, dim=-1).indices
            rank = ((parents[:, :, None] == parents[:, None, :]) & torch.ones(nodes, nodes, device="cuda").tril(-1).bool()).sum(-1) % 16
            tokens = guess.gather(1, (parents.long() + 1)[..., None].expand(-1, -1, 16)).gather(2, rank[..., None])[..., 0]
            draft = None
        else:
            parents = None
            draft = torch.softmax(logits[:, :nodes] + 0.7 * normal(batch, nodes, vocab), -1)
            tokens = (draft / torch.empty_like(draft).exponential_(generator=gen)).argmax(-1)
        return dict(kind=kind, target=torch.softmax(logits, -1), draft=draft, tokens=tokens.int(), parents=parents,
                    counts=ints(_counts(case)) if case["tree"] else None, accept=uniform(batch, nodes), sample=uniform(batch))
    lengths = _lengths(case)
    state = dict(kind=kind, lengths=ints(lengths), longest=case["longest"])
    if kind in ("write", "commit"):
        tokens = case["tokens"] if kind == "write" else case["nodes"]
        dtype = torch.bfloat16 if case["bf16"] else torch.float32
        state["page"], state["table"], k, v = _pool(case, case["longest"] + tokens, torch.uint8, gen)
        state["k_pool"], state["v_pool"] = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
        state["k_scales"], state["v_scales"] = (torch.zeros(k.shape[:3], dtype=torch.uint8, device="cuda") for _ in range(2))
        # keys have channels that are larger than the rest
        loud = 1 + 15 * (uniform(case["heads"], case["dim"]) < 0.02)
        state["k"] = (normal(batch, tokens, case["heads"], case["dim"]) * loud).to(dtype)
        state["v"] = normal(batch, tokens, case["heads"], case["dim"]).to(dtype)
        state["tokens"] = tokens
        if kind == "commit":
            accepted = ints(_accepted(case))
            order = torch.sort(uniform(batch, tokens).argsort(-1)[:, :min(8, tokens)], -1).values.int()
            order = order.sort(-1).values
            path = torch.full((batch, tokens), -1, dtype=torch.int32, device="cuda")
            path[:, :order.shape[1]] = order
            state["accepted"] = accepted
            state["path"] = torch.where(torch.arange(tokens, device="cuda") < accepted[:, None], path, torch.full_like(path, -1))
        return state
    nodes, dim, hq = case["nodes"], case["dim"], case["q_heads"]
    state["page"], state["table"], k, v = _pool(case, case["longest"] + nodes, torch.bfloat16, gen)
    state["k_scales"] = state["v_scales"] = None
    k.normal_(generator=gen)
    v.normal_(generator=gen)
    if case["eight"]:
        (k, state["k_scales"]), (v, state["v_scales"]) = _quantise(k), _quantise(v)
        k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
    state["k_pool"], state["v_pool"] = k, v
    state["q"] = normal(batch, nodes, hq, dim).bfloat16()
    state["gate"] = normal(batch, nodes, hq, dim).bfloat16() if case["gate"] else None
    state["parents"] = (uniform(batch, nodes) * torch.arange(1, nodes + 1, device="cuda")).int() - 1 if case["tree"] else None
    state["counts"] = ints(_counts(case)) if case["tree"] else None
    state["out"] = torch.zeros_like(state["q"])
    return state


# ---- the operators' definitions in elementary operations -----------------------------------------------------

def _write_plain(s):
    slots = s["lengths"].long()[:, None] + torch.arange(s["tokens"], device="cuda")
    rows = _rows(s, slots)
    heads, dim = s["k"].shape[2:]
    k_pool, v_pool = (s[p].view(torch.uint8).view(-1, heads, dim) for p in ("k_pool", "v_pool"))
    k_scales, v_scales = s["k_scales"].view(-1, heads), s["v_scales"].view(-1, heads)
    k_pool[rows], k_scales[rows] = _quantise(s["k"])
    v_pool[rows], v_scales[rows] = _quantise(s["v"])
    if s["kind"] == "commit":
        # the rows of the path, in order, to the first slots; the others stay where they are
        kept = torch.arange(s["tokens"], device="cuda") < s["accepted"][:, None]
        source = rows.gather(1, torch.where(kept, s["path"].long(), torch.arange(s["tokens"], device="cuda")))
        k_pool[rows], k_scales[rows] = k_pool[source], k_scales[source]
        v_pool[rows], v_scales[rows] = v_pool[source], v_scales[source]
    return [_values(k_pool[rows], k_scales[rows]).to(s["k"].dtype), _values(v_pool[rows], v_scales[rows]).to(s["v"].dtype)]


def _ancestors(parents):
    """[B, N, N]: whether node j is node i or one of its ancestors: the inverse of (I - parent matrix)."""
    n = parents.shape[1]
    one = torch.eye(n, device="cuda").expand(parents.shape[0], n, n)
    child = (parents[:, :, None] == torch.arange(n, device="cuda")).float()
    return torch.linalg.solve_triangular(one - child, one, upper=False) > 0.5


def _attend_plain(s):
    q = s["q"].float()
    batch, nodes, hq, dim = q.shape
    hkv, longest = s["k_pool"].shape[2], s["longest"] + nodes
    slots = torch.arange(longest, device="cuda").expand(batch, longest)
    rows = _rows(s, slots)
    if s["k_scales"] is None:
        k, v = (s[p].view(-1, hkv, dim)[rows].float() for p in ("k_pool", "v_pool"))
    else:
        k, v = (_values(s[p].view(torch.uint8).view(-1, hkv, dim)[rows], s[c].view(-1, hkv)[rows])
                for p, c in (("k_pool", "k_scales"), ("v_pool", "v_scales")))
    counts = s["counts"] if s["counts"] is not None else torch.full((batch,), nodes, device="cuda")
    parents = s["parents"] if s["parents"] is not None else torch.arange(-1, nodes - 1, device="cuda").expand(batch, nodes)
    offset = slots - s["lengths"][:, None]
    seen = _ancestors(parents).gather(2, offset.clamp(0, nodes - 1)[:, None, :].expand(batch, nodes, longest))
    seen = ((offset < 0)[:, None, :] | (seen & (offset >= 0)[:, None, :])) & (offset < counts[:, None])[:, None, :]
    grouped = q.view(batch, nodes, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, dim)
    scores = torch.matmul(grouped, k.permute(0, 2, 3, 1)) / math.sqrt(dim)
    scores = scores.view(batch, hkv, nodes, hq // hkv, longest).masked_fill(~seen[:, None, :, None, :], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(batch, hkv, -1, longest), v.permute(0, 2, 1, 3))
    out = out.view(batch, hkv, nodes, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(batch, nodes, hq, dim)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    return torch.where((torch.arange(nodes, device="cuda") < counts[:, None])[:, :, None, None], out, 0.0).bfloat16()


def _verify_plain(s):
    target, tokens = s["target"], s["tokens"].long()
    batch, nodes = tokens.shape
    vocab = target.shape[2]
    index = torch.arange(nodes, device="cuda")
    counts = s["counts"].long() if s["counts"] is not None else torch.full((batch,), nodes, device="cuda")
    alive = index < counts[:, None]
    each = torch.arange(batch, device="cuda")
    parents = s["parents"].long() if s["parents"] is not None else index.expand(batch, nodes) - 1
    p = target[each[:, None], parents + 1, tokens].double()
    u = s["accept"].double()
    if s["draft"] is not None:
        q = s["draft"][each[:, None], index, tokens].double()
        taken = ((u * q < p) & alive).cumprod(-1).bool()
        accepted = taken.sum(-1)
        last = accepted - 1
    else:
        earlier = (parents[:, :, None] == parents[:, None, :]) & (index[:, None] > index)
        again = (earlier & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
        left = 1 - (earlier * torch.where(again, 0.0, p)[:, None, :]).sum(-1)
        good = (u * left < p) & ~again & alive
        good = good & ~(earlier & good[:, None, :]).any(-1)
        taken = torch.matmul(_ancestors(parents).float(), (~good).float()[..., None])[..., 0] < 0.5
        accepted = taken.sum(-1)
        last = torch.where(taken, index, -1).amax(-1)
    path = torch.where(taken, index, nodes).sort(-1).values
    path = torch.where(path < nodes, path, -1)
    row = target[each, last + 1].double()
    if s["draft"] is not None:
        rest = (row - s["draft"][each, accepted.clamp(max=nodes - 1)].double()).clamp(min=0)
        rest = torch.where((accepted < counts)[:, None], rest, row)
    else:
        tried = (parents == last[:, None]) & alive
        keep = torch.ones(batch, vocab + 1, dtype=torch.float64, device="cuda").scatter(1, torch.where(tried, tokens, vocab), 0.0)
        rest = row * keep[:, :vocab]
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, row)
    sums = rest.cumsum(-1)
    total = sums[:, -1:]
    drawn = torch.searchsorted(sums, s["sample"].double()[:, None] * total, right=True).clamp(max=vocab - 1)[:, 0]
    drawn = torch.where((total[:, 0] > 0) & torch.isfinite(total[:, 0]), drawn, -1)
    out = torch.cat([torch.where(path >= 0, tokens.gather(1, path.clamp(min=0)), -1), torch.full((batch, 1), -1, device="cuda")], 1)
    out[each, accepted] = drawn
    return [accepted.int(), path.int(), out.int()]


def run(state):
    s = state
    if not own:
        return {"write": _write_plain, "commit": _write_plain, "attend": _attend_plain, "verify": _verify_plain}[s["kind"]](s)
    from pluto_b200 import layers
    if s["kind"] in ("write", "commit"):
        cache = s["k_pool"], s["v_pool"], s["k_scales"], s["v_scales"]
        layers.kv8_append(s["k"], s["v"], *cache, s["lengths"], block_table=s["table"])
        if s["kind"] == "commit":
            layers.kv_keep(s["k_pool"], s["v_pool"], s["lengths"], s["path"], s["accepted"], block_table=s["table"],
                           k_scales=s["k_scales"], v_scales=s["v_scales"])
        return list(layers.kv8_read(*cache, s["lengths"], s["tokens"], block_table=s["table"], dtype=s["k"].dtype))
    if s["kind"] == "attend":
        return layers.gqa_tree_decode(s["q"], s["k_pool"], s["v_pool"], s["lengths"], s["longest"], parents=s["parents"],
                                      counts=s["counts"], block_table=s["table"], k_scales=s["k_scales"], v_scales=s["v_scales"],
                                      gate=s["gate"], round_to_bfloat16=False, out=s["out"])
    result = layers.verify_drafts(s["target"], s["tokens"], s["accept"], s["sample"], parents=s["parents"], counts=s["counts"],
                                  draft_probs=s["draft"])
    return [result.accepted, result.path, result.tokens]


def work(case):
    if case["kind"] == "verify":
        # the row that the last token is drawn from, and the draft's beside it where the drafts were sampled
        rows = case["batch"] * (1 if case["tree"] else 2)
        return dict(bytes=4 * rows * case["vocab"] + 24 * case["batch"] * case["nodes"], flops=3 * rows * case["vocab"])
    heads, dim = case.get("heads", case.get("kv_heads")), case["dim"]
    if case["kind"] == "attend":
        cached = sum(n + 1 for n in _lengths(case))
        drafts = sum(_counts(case))
        row = 2 * heads * (dim + 1 if case["eight"] else 2 * dim)
        seen = sum(n * (length + 1) for n, length in zip(_counts(case), _lengths(case)))
        return dict(bytes=row * (cached + drafts - case["batch"]) + drafts * case["q_heads"] * dim * (6 if case["gate"] else 4),
                    flops=4 * dim * case["q_heads"] * seen)
    tokens = case["batch"] * (case["tokens"] if case["kind"] == "write" else case["nodes"])
    element = 2 if case["bf16"] else 4
    moved = sum(_accepted(case)) if case["kind"] == "commit" else 0
    # rows in, codes out, codes in again, values out
    return dict(bytes=2 * heads * (tokens * (2 * element * dim + 2 * (dim + 1)) + 2 * moved * (dim + 1)), flops=8 * heads * dim * tokens)


def exact(case, seed):
    """The result in 64 bits, from the definitions alone."""
    s = prepare(case, seed)
    if case["kind"] in ("write", "commit"):
        def power(n):
            return ((n.long() + 1023) << 52).view(torch.float64)

        def floor_log2(x):
            return ((x.contiguous().view(torch.int64) >> 52) & 0x7ff) - 1023

        def held(x):
            x = x.double()
            largest = x.abs().amax(-1, keepdim=True)
            n = floor_log2(largest).clamp(min=-200) - 9
            n = torch.where(448 * power(n) < largest, n + 1, n)
            n = torch.where(448 * power(n) < largest, n + 1, n).clamp(min=-127)
            y = x / power(n)
            step = power(floor_log2(y.abs().clamp(min=2.0 ** -6)) - 3)
            return torch.round(y / step) * step * power(n)
        k, v = held(s["k"]), held(s["v"])
        if case["kind"] == "commit":
            for b, n in enumerate(s["accepted"].tolist()):
                nodes = s["path"][b, :n].long()
                k[b, :n], v[b, :n] = k[b, nodes].clone(), v[b, nodes].clone()
        return [k, v]
    if case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["q_heads"] // case["kv_heads"]
        for b, (length, count) in enumerate(zip(_lengths(case), _counts(case))):
            where = torch.arange(length + count, device="cuda")
            pages, inside = s["table"][b, where // s["page"]].long(), where % s["page"]
            k, v = s["k_pool"][pages, inside].double(), s["v_pool"][pages, inside].double()
            if case["eight"]:
                k, v = (x * ((n[pages, inside].long() - 127 + 1023) << 52).view(torch.float64)[..., None]
                        for x, n in ((k, s["k_scales"]), (v, s["v_scales"])))
            seen = torch.zeros(count, length + count, dtype=torch.bool)
            seen[:, :length] = True
            parents = s["parents"][b].tolist() if case["tree"] else list(range(-1, count - 1))
            for i in range(count):
                seen[i, length + i] = True
                if parents[i] >= 0:
                    seen[i, length:] |= seen[parents[i], length:]
            seen = seen.cuda()
            for h in range(case["kv_heads"]):
                q = s["q"][b, :count, h * group:(h + 1) * group].double()
                scores = torch.einsum("ngd,td->ngt", q, k[:, h]) / math.sqrt(case["dim"])
                weights = torch.softmax(scores.masked_fill(~seen[:, None, :], -math.inf), -1)
                out[b, :count, h * group:(h + 1) * group] = torch.einsum("ngt,td->ngd", weights, v[:, h])
        return out * torch.sigmoid(s["gate"].double()) if case["gate"] else out
    accepted, paths, tokens = [], [], []
    drafted, u_all, u_last = s["tokens"].tolist(), s["accept"].double().tolist(), s["sample"].double().tolist()
    for b, count in enumerate(_counts(case)):
        node, path, tried, refused = -1, [], set(), None
        parents = s["parents"][b].tolist() if case["tree"] else list(range(-1, count - 1))
        i, left = 0, 1.0
        while i < count:
            if parents[i] == node:
                token = drafted[b][i]
                p = float(s["target"][b, node + 1, token])
                if case["tree"]:
                    good = token not in tried and u_all[b][i] * left < p
                else:
                    good = u_all[b][i] * float(s["draft"][b, i, token]) < p
                if good:
                    node, tried, left = i, set(), 1.0
                    path.append(i)
                else:
                    refused = i
                    left -= 0.0 if token in tried else p
                    tried.add(token)
                    if not case["tree"]:
                        break
            i += 1
        row = s["target"][b, node + 1].double()
        rest = row.clone()
        if case["tree"]:
            rest[list(tried)] = 0.0
        elif refused is not None:
            rest = (row - s["draft"][b, refused].double()).clamp(min=0)
        if not float(rest.sum()) > 0:
            rest = row
        sums = torch.cumsum(rest.cpu(), 0)
        drawn = int((sums <= u_last[b] * float(sums[-1])).sum())
        accepted.append(len(path))
        paths.append(path + [-1] * (case["nodes"] - len(path)))
        tokens.append([drafted[b][i] for i in path] + [drawn] + [-1] * (case["nodes"] - len(path)))
    return [torch.tensor(x, dtype=torch.int32) for x in (accepted, paths, tokens)]
