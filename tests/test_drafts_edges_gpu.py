"""Drafted tokens and the 8-bit cache at the edges of their ranges, against plain 64-bit models."""
import math

import pytest
import torch

from drafts_double import tree_attention
from pluto_b200 import PlutoStatusError, _capi
from pluto_b200.layers import draft_prepare, gqa_tree_decode, kv8_append, kv8_read, kv_keep, verify_drafts

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")
EIGHT = torch.float8_e4m3fn
# (nodes, query heads, KV heads, width): up to 8 and 16 rows per KV head, up to 128, more than 128
SHAPES = [(1, 10, 2, 128), (3, 4, 4, 64), (1, 6, 1, 256), (3, 10, 2, 128), (20, 10, 2, 128), (30, 4, 4, 64), (20, 6, 1, 256), (40, 20, 4, 128), (70, 6, 3, 64)]


def random(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return gen, lambda *s: torch.randn(*s, device="cuda", generator=gen)


def values(codes, scales):
    """The float64 values of 8-bit rows."""
    power = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64, device="cuda"), scales.int() - 127)
    return codes.double() * torch.where(scales == 255, math.nan, power)[..., None]


@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
@pytest.mark.parametrize("k_powers,v_powers", [
    ([-20, -16, -15, -3, 0, 7, 8, 12], [0]), ([0], [-40, -16, 0, 7, 8, 20]), ([-16, 0, 8], [-90, -17, 9, 90]), ([-1], [-127, -30]), ([0], [-12, -9])])
def test_row_scales_that_fp16_does_not_hold(nodes, hq, hkv, dim, k_powers, v_powers):
    gen, rnd = random(nodes + dim)
    prefix, rows = 333, 333 + nodes
    pick = lambda powers: torch.tensor(powers, device="cuda")[torch.randint(0, len(powers), (1, rows, hkv), device="cuda", generator=gen)]  # noqa: E731
    kn, vn = pick(k_powers), pick(v_powers)
    k = (rnd(1, rows, hkv, dim) * 2.0 ** -kn.clamp(min=-3)[..., None]).to(EIGHT)   # keys near 1, or smaller
    v = (rnd(1, rows, hkv, dim) * 16).to(EIGHT)
    v.view(torch.uint8)[0, 5] = 0
    vn[0, 5] = -127                                                                # a row of zeros
    k_scales, v_scales = (kn + 127).to(torch.uint8), (vn + 127).to(torch.uint8)
    q = rnd(1, nodes, hq, dim).bfloat16()
    parents = ((torch.rand(1, nodes, device="cuda", generator=gen) * torch.arange(1, nodes + 1, device="cuda")).int() - 1)
    got, lse = gqa_tree_decode(q, k, v, torch.tensor([prefix], **INT), prefix, parents=parents, k_scales=k_scales, v_scales=v_scales,
                               round_to_bfloat16=False, want_lse=True)
    want, mean, want_lse = tree_attention(q[0].double(), values(k, k_scales)[0], values(v, v_scales)[0], prefix, parents[0].tolist())
    # Weights carry fp16's 11 bits (bf16 outputs round once: 2^-8), as long as they are normal: they are taken times their
    # row's 2^n relative to the largest 2^n, so below 2^-14 they are off by up to 2^-25 of the largest 2^n (times the row's
    # own 2^n where that went into its codes, n <= 7), against a sum of weights of at least 1.
    group = hq // hkv
    lost = 2.0 ** -25 * 2.0 ** max(max(v_powers), 0) * (v.double().abs() * 2.0 ** vn.clamp(0, 7)[..., None]).sum(1)[0].repeat_interleave(group, 0)
    bound = mean * 2.0 ** -11 * 1.01 + lost + 2.0 ** -8 * want.abs() * 1.01 + 2.0 ** -20 * mean
    off = (got[0].double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    assert (lse[0].double() - want_lse).abs().max().item() < 2e-5 * max(1.0, want_lse.abs().max().item())
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("store", [EIGHT, torch.bfloat16])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_rows_that_are_not_finite_in_the_prefix(store, nodes, hq, hkv, dim):
    """They reach every node of their sequence and KV head, and nothing else."""
    gen, rnd = random(dim)
    k, v, q, at = rnd(3, 200, hkv, dim), rnd(3, 200, hkv, dim), rnd(3, nodes, hq, dim).bfloat16(), torch.tensor([100, 120, 99], **INT)

    def run(k, v):
        if store != EIGHT:
            return gqa_tree_decode(q, k.to(store), v.to(store), at, 120)
        rows = [torch.zeros(3, 200, hkv, dim, dtype=store, device="cuda") for _ in range(2)]
        rows += [torch.zeros(3, 200, hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k, v, *rows)
        return gqa_tree_decode(q, rows[0], rows[1], at, 120, k_scales=rows[2], v_scales=rows[3])
    clean, group = run(k, v), hq // hkv
    assert torch.isfinite(clean).all()
    for bad_k, bad_v, token in ((math.nan, None, 0), (None, math.nan, 17), (None, math.inf, 99), (math.inf, None, 63)):
        kk, vv = k.clone(), v.clone()
        if bad_k is not None:
            kk[1, token, hkv - 1] = bad_k
        if bad_v is not None:
            vv[1, token, hkv - 1] = bad_v
        got = run(kk, vv)
        hit = got[1, :, (hkv - 1) * group:]
        assert not torch.isfinite(hit).any()
        got[1, :, (hkv - 1) * group:] = clean[1, :, (hkv - 1) * group:]
        assert torch.equal(got, clean)
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("kind", ["fp32", "odd", "slice"])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_gates_of_other_types_and_strides(nodes, hq, hkv, dim, kind):
    gen, rnd = random(nodes)
    k, v, q = rnd(2, 150, hkv, dim).bfloat16(), rnd(2, 150, hkv, dim).bfloat16(), rnd(2, nodes, hq, dim).bfloat16()
    if kind == "fp32":
        gate = rnd(2, nodes, hq, dim)
    elif kind == "odd":
        gate = rnd(2, nodes, hq, dim + 1).bfloat16()[..., 1:]
    else:
        gate = rnd(2, nodes, hq + 3, 2, dim).bfloat16()[:, :, 2:hq + 2, 1]
    at = torch.tensor([150 - nodes, 11], **INT)
    got = gqa_tree_decode(q, k, v, at, 150, gate=gate, round_to_bfloat16=False)
    for b in range(2):
        n = int(at[b])
        want, mean, _ = tree_attention(q[b].double(), k[b, :n + nodes].double(), v[b, :n + nodes].double(), n, list(range(-1, nodes - 1)))
        factor = torch.sigmoid(gate[b].double())
        # weights rounded to bf16 (2^-8 of a mean of |v|) or better, the result rounded once
        assert ((got[b].double() - want * factor).abs() <= (mean * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -8 * 1.01 * want.abs()) * factor + 1e-6).all()
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("nodes,dim,hkv,group", [(1, 64, 72, 1), (2, 128, 65, 2), (1, 128, 64, 1), (2, 64, 3, 2), (1, 256, 5, 3), (9, 64, 70, 1)])
def test_many_and_odd_numbers_of_kv_heads(nodes, dim, hkv, group):
    """Heads side by side and one after the other; 8-bit scales at odd addresses."""
    gen, rnd = random(hkv)
    wide = hkv + 3
    rows = [torch.zeros(4, 150, wide, dim, dtype=EIGHT, device="cuda") for _ in range(2)]
    rows += [torch.zeros(4, 150, wide, dtype=torch.uint8, device="cuda") for _ in range(2)]
    kv8_append(rnd(4, 150, wide, dim), rnd(4, 150, wide, dim), *rows)
    shard = [r[:, :, 3:] for r in rows]
    k, v = (x[:, :, 3:].double() for x in kv8_read(*rows, torch.zeros(4, **INT), 150, dtype=torch.float32))
    at, q = torch.tensor([149 - nodes, 0, 77, 16], **INT), rnd(4, nodes, hkv * group, dim).bfloat16()
    got = gqa_tree_decode(q, shard[0], shard[1], at, 149, k_scales=shard[2], v_scales=shard[3], round_to_bfloat16=False)
    for b in range(4):
        n = int(at[b])
        want, mean, _ = tree_attention(q[b].double(), k[b, :n + nodes], v[b, :n + nodes], n, list(range(-1, nodes - 1)))
        assert ((got[b].double() - want).abs() <= mean * (2.0 ** -11 * 1.01 + 2.0 ** -20) + 2.0 ** -8 * 1.01 * want.abs() + 1e-6).all()
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("store", [EIGHT, torch.bfloat16])
@pytest.mark.parametrize("nodes,hq,hkv,dim,longest", [(61, 40, 8, 128, 4000), (61, 40, 8, 128, 200), (40, 20, 4, 64, 3000), (20, 40, 8, 128, 3000), (20, 24, 4, 256, 2000), (3, 10, 2, 128, 3000)])
def test_many_calls_agree(store, nodes, hq, hkv, dim, longest):
    """The order of every sum is fixed, so calls repeat bit for bit whatever the warps' timing."""
    gen, rnd = random(nodes + longest)
    k, v = (rnd(8, longest + nodes, hkv, dim) for _ in range(2))
    scales = [None, None]
    if store == EIGHT:
        rows = [torch.zeros(8, longest + nodes, hkv, dim, dtype=EIGHT, device="cuda") for _ in range(2)]
        rows += [torch.zeros(8, longest + nodes, hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k * 2.0 ** torch.randint(-4, 4, k.shape[:3] + (1,), device="cuda", generator=gen), v * 2.0 ** torch.randint(-4, 4, v.shape[:3] + (1,), device="cuda", generator=gen), *rows)
        k, v, *scales = rows
    else:
        k, v = k.bfloat16(), v.bfloat16()
    q = rnd(8, nodes, hq, dim).bfloat16()
    at = torch.randint(0, longest + 1, (8,), device="cuda", generator=gen).int()
    counts = torch.randint(nodes // 2, nodes + 1, (8,), device="cuda", generator=gen).int()
    out = torch.zeros_like(q)
    call = lambda: gqa_tree_decode(q, k, v, at, longest, counts=counts, k_scales=scales[0], v_scales=scales[1], out=out)  # noqa: E731
    first, off = call().clone(), torch.zeros((), device="cuda")
    for _ in range(1500):
        off += (call() != first).any()
    assert off.item() == 0 and _capi.kernel_status() == 0


@pytest.mark.parametrize("store", [EIGHT, torch.bfloat16])
def test_short_pieces_of_units_agree(store):
    """Many ragged sequences, cut so that some pieces hold a tile or two: calls repeat bit for bit."""
    gen, rnd = random(5)
    off = torch.zeros((), device="cuda")
    for turn in range(24):
        batch, nodes, longest = (24, 16)[turn % 2], (31, 40, 62)[turn % 3], (2664, 900, 300)[turn % 3]
        k, v = (rnd(batch, longest + nodes, 12, 128).to(store) for _ in range(2))
        scales = [torch.randint(124, 129, k.shape[:3], device="cuda", generator=gen).to(torch.uint8) if store == EIGHT else None for _ in range(2)]
        q = rnd(batch, nodes, 60, 128).bfloat16()
        at = torch.randint(0, longest + 1, (batch,), device="cuda", generator=gen).int()
        counts = torch.randint(0, nodes + 1, (batch,), device="cuda", generator=gen).int()
        out = torch.zeros_like(q)
        call = lambda: gqa_tree_decode(q, k, v, at, longest, counts=counts, k_scales=scales[0], v_scales=scales[1], out=out)  # noqa: E731
        first = call().clone()
        for _ in range(60):
            off += (call() != first).any()
    assert off.item() == 0 and _capi.kernel_status() == 0


@pytest.mark.parametrize("nodes", [1, 20, 60])
def test_no_sequence_has_a_node(nodes):
    gen, rnd = random(2)
    k, q = rnd(3, 100, 2, 128).bfloat16(), rnd(3, nodes, 10, 128).bfloat16()
    out = torch.full_like(q, 3.0)
    for counts in ([0, 0, 0], [0, 1, 0]):
        gqa_tree_decode(q, k, k, torch.tensor([40, 0, 7], **INT), 40, counts=torch.tensor(counts, **INT), out=out)
        assert (out[0] == 3).all() and (out[2] == 3).all() and (out[1, 1:] == 3).all()
    assert torch.equal(out[1, 0].view(2, 5, 128), k[1, 0][:, None].expand(2, 5, 128))   # one key: its value
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("store", [EIGHT, torch.bfloat16])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 32, 64, 10])
def test_bad_pages_in_the_prefix(store, nodes, hq, hkv, dim, page):
    """Pages outside the pool are reported and read as zeros; the other sequences are as with good ones."""
    gen, rnd = random(page)
    blocks = -(-(210 + nodes) // page)
    table = torch.randperm(3 * blocks, device="cuda", generator=gen).int().view(3, blocks)
    k, v = (rnd(3 * blocks, page, hkv, dim).to(store) for _ in range(2))
    scales = [torch.full((3 * blocks, page, hkv), 127, dtype=torch.uint8, device="cuda") if store == EIGHT else None for _ in range(2)]
    q, at = rnd(3, nodes, hq, dim).bfloat16(), torch.tensor([210, 205, 190], **INT)
    call = lambda t, k, v: gqa_tree_decode(q, k, v, at, 210, block_table=t, k_scales=scales[0], v_scales=scales[1])  # noqa: E731
    good = call(table, k, v)
    assert _capi.kernel_status() == 0
    for bad in (-1, 3 * blocks, 2 ** 31 - 1, -2 ** 31):
        wrong = table.clone()
        wrong[1, 1], wrong[1, 128 // page] = bad, bad
        got = call(wrong, k, v)
        assert _capi.kernel_status() & 0xff == 3
        zeros = [x.clone() for x in (k, v)]
        for x in zeros:
            x.view(torch.uint8)[table[1, 1].item()] = 0
            x.view(torch.uint8)[table[1, 128 // page].item()] = 0
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
        want = call(table, *zeros)
        if store == EIGHT:
            # The rows that read as zeros have scale byte 0, those of the pool of zeros 127.  Where a range of the line holds nothing
            # else, its weights are relative to another power of two, and the merge's 2^(m_c - m) differs by the 2^-22 that
            # ex2.approx is off: 2^-20 of a result below max|v| (448 at scale 2^0, here below 8), then its rounding to bf16, which
            # may fall to the other side: a step, 2^-7 of the result.
            assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 8 * 2.0 ** -20).all()
        else:
            assert torch.equal(got, want)
    assert _capi.kernel_status() == 0


def test_pools_beyond_32_bits():
    """Pages whose rows lie more than 2^32 elements into the pool."""
    gen, rnd = random(4)
    pages, heads, dim = 270000, 8, 128
    pools = [torch.empty(pages, 16, heads, dim, dtype=EIGHT, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, 16, heads, dtype=torch.uint8, device="cuda") for _ in range(2)]
    assert pools[0].numel() > 2 ** 32
    for nodes in (1, 9, 60):
        capacity = 64 + nodes
        blocks = -(-capacity // 16)
        table = torch.arange(pages - 1, pages - 1 - 2 * blocks, -1, **INT).view(2, blocks)
        k, v, q = rnd(2, capacity, heads, dim), rnd(2, capacity, heads, dim), rnd(2, nodes, 16, dim).bfloat16()
        kv8_append(k, v, *pools, *scales, block_table=table)
        small = [torch.zeros(2, capacity, heads, dim, dtype=EIGHT, device="cuda") for _ in range(2)]
        small += [torch.zeros(2, capacity, heads, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k, v, *small)
        zero = torch.zeros(2, **INT)
        for a, b in zip(kv8_read(*pools, *scales, zero, capacity, block_table=table), kv8_read(*small, zero, capacity)):
            assert torch.equal(a, b)
        at = torch.tensor([64, 50], **INT)
        got = gqa_tree_decode(q, *pools, at, 64, block_table=table, k_scales=scales[0], v_scales=scales[1])
        assert torch.equal(got, gqa_tree_decode(q, small[0], small[1], at, 64, k_scales=small[2], v_scales=small[3]))
        path, accepted = torch.full((2, nodes), -1, **INT), torch.tensor([1, 0], **INT)
        path[0, 0] = nodes - 1
        kv_keep(*pools, at, path, accepted, block_table=table, k_scales=scales[0], v_scales=scales[1])
        kv_keep(*small[:2], at, path, accepted, k_scales=small[2], v_scales=small[3])
        for a, b in zip(kv8_read(*pools, *scales, zero, capacity, block_table=table), kv8_read(*small, zero, capacity)):
            assert torch.equal(a, b)
    assert _capi.kernel_status() == 0


def test_a_captured_speculative_step():
    """Prepare, attention, verification and the cache step in one graph, replayed on changed inputs and on another stream."""
    gen, rnd = random(12)
    B, N, hq, hkv, dim, vocab = 3, 6, 10, 2, 128, 999
    parents = torch.tensor([[-1, 0, 0, 1, -1, 2]] * B, **INT)
    state = dict(q=rnd(B, N, hq, dim).bfloat16(), k=rnd(B, N, hkv, dim).bfloat16(), v=rnd(B, N, hkv, dim).bfloat16(),
                 at=torch.tensor([40, 3, 77], **INT), target=torch.softmax(rnd(B, N + 1, vocab) * 3, -1),
                 tokens=torch.randint(0, vocab, (B, N), device="cuda", generator=gen).int(),
                 u=torch.zeros(B, N, device="cuda"), u_last=torch.rand(B, device="cuda", generator=gen))
    norm, cache = rnd(dim) * 0.1, lambda: dict(  # noqa: E731
        k_pool=torch.zeros(B, 120, hkv, dim, dtype=EIGHT, device="cuda"), v_pool=torch.zeros(B, 120, hkv, dim, dtype=EIGHT, device="cuda"),
        k_scales=torch.zeros(B, 120, hkv, dtype=torch.uint8, device="cuda"), v_scales=torch.zeros(B, 120, hkv, dtype=torch.uint8, device="cuda"))

    def step(s, pool):
        queries = draft_prepare(s["q"], s["k"], s["v"], norm, norm, s["at"], **pool, rotary_dim=64, parents=parents)
        out = gqa_tree_decode(queries, pool["k_pool"], pool["v_pool"], s["at"], 100, parents=parents, k_scales=pool["k_scales"], v_scales=pool["v_scales"])
        verdict = verify_drafts(s["target"], s["tokens"], s["u"], s["u_last"], parents=parents)
        kv_keep(pool["k_pool"], pool["v_pool"], s["at"], verdict.path, verdict.accepted, k_scales=pool["k_scales"], v_scales=pool["v_scales"])
        return (out, *verdict, *kv8_read(pool["k_pool"], pool["v_pool"], pool["k_scales"], pool["v_scales"], s["at"], N))
    captured_pool, eager_pool = cache(), cache()
    step(state, cache())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(state, captured_pool)
    other = torch.cuda.Stream()
    for turn in range(4):
        state["q"].copy_(rnd(B, N, hq, dim))
        state["k"].copy_(rnd(B, N, hkv, dim))
        state["at"].copy_(torch.randint(0, 100, (B,), device="cuda", generator=gen).int())
        state["u"].copy_(torch.rand(B, N, device="cuda", generator=gen) * 1e-3)
        torch.cuda.synchronize()
        with torch.cuda.stream(other if turn % 2 else torch.cuda.current_stream()):
            graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outputs, step(state, eager_pool)):
            assert torch.equal(got, want)
    assert _capi.kernel_status() == 0


def test_a_report_that_nobody_has_read_does_not_touch_later_calls():
    """A bad draft is reported; the attention calls behind it are those of a healthy status word."""
    gen, rnd = random(6)
    calls = []
    for nodes, hq, hkv, dim, store in ((61, 40, 8, 128, EIGHT), (40, 24, 4, 256, torch.bfloat16), (1, 40, 8, 128, EIGHT), (30, 12, 12, 64, torch.bfloat16)):
        q, at = rnd(4, nodes, hq, dim).bfloat16(), torch.tensor([9000, 100, 8000, 4000], **INT)
        rows = [rnd(4, 9100, hkv, dim).to(store) for _ in range(2)]
        scales = [torch.full((4, 9100, hkv), 127, dtype=torch.uint8, device="cuda") if store == EIGHT else None for _ in range(2)]
        calls.append(lambda q=q, r=rows, s=scales, at=at: gqa_tree_decode(q, r[0], r[1], at, 9000, k_scales=s[0], v_scales=s[1]))
    want = [call() for call in calls]
    assert _capi.kernel_status() == 0
    verify_drafts(torch.full((1, 2, 4), 0.25, device="cuda"), torch.full((1, 1), 7, **INT), torch.zeros(1, 1, device="cuda"), torch.zeros(1, device="cuda"))
    for _ in range(20):
        for call, clean in zip(calls, want):
            assert torch.equal(call(), clean)
    assert _capi.kernel_status() & 0xff == 5 and _capi.kernel_status() == 0


def test_tensors_elsewhere_are_refused():
    k = torch.zeros(2, 16, 2, 64, dtype=EIGHT, device="cuda")
    s = torch.zeros(2, 16, 2, dtype=torch.uint8, device="cuda")
    x, at = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, **INT)
    for call in (lambda: kv8_append(x.cpu(), x.cpu(), k, k, s, s, at), lambda: kv8_append(x, x, k, k, s, s.cpu(), at),
                 lambda: kv8_append(x, x, k, k.cpu(), s, s, at), lambda: kv8_append(x, x, k, k, s, s, at.cpu()),
                 lambda: kv8_read(k, k, s, s, at.cpu(), 1), lambda: kv_keep(k, k, at, at[:, None], at.cpu(), k_scales=s, v_scales=s),
                 lambda: gqa_tree_decode(x, k, k, at, 8, k_scales=s, v_scales=s, counts=at.cpu()),
                 lambda: gqa_tree_decode(x.cpu(), k, k, at, 8, k_scales=s, v_scales=s),
                 lambda: gqa_tree_decode(x, k, k, at, 8, k_scales=s, v_scales=s, out=x.cpu()),
                 lambda: gqa_tree_decode(x, k, k, at, 8, k_scales=s, v_scales=s, gate=x.cpu()),
                 lambda: gqa_tree_decode(x, k, k, at, 8, k_scales=s, v_scales=s, workspace=torch.empty(1 << 24, dtype=torch.uint8)),
                 lambda: verify_drafts(torch.zeros(2, 2, 5, device="cuda"), at[:, None], torch.zeros(2, 1), torch.zeros(2, device="cuda")),
                 lambda: verify_drafts(torch.zeros(2, 2, 5), at[:, None], torch.zeros(2, 1, device="cuda"), torch.zeros(2, device="cuda")),
                 lambda: verify_drafts(torch.zeros(2, 2, 5, device="cuda"), at[:, None], torch.zeros(2, 1, device="cuda"), torch.zeros(2, device="cuda"),
                                       draft_probs=torch.zeros(2, 1, 5))):
        with pytest.raises(PlutoStatusError):
            call()
    assert _capi.kernel_status() == 0
