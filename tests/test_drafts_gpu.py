"""Drafted tokens and the 8-bit cache against plain 64-bit models (tests/drafts_double.py)."""
import math

import pytest
import torch

from drafts_double import e8m0_rows, tree_attention, verify
from pluto_b200 import PlutoStatusError, _capi
from pluto_b200.layers import (CachedAttentionStep, CachedDraftStep, FullAttentionParameters, KeyValueCache, draft_prepare,
                               gqa_decode, gqa_tree_decode, kv8_append, kv8_read, kv_keep, verify_drafts)

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


def random(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return gen, lambda *s: torch.randn(*s, device="cuda", generator=gen)


def pages_of(batch, capacity, page, gen):
    """Block table with the sequences' pages scattered over the pool, or None and one page per sequence."""
    if not page:
        return None, batch, capacity
    blocks = -(-capacity // page)
    table = torch.randperm(batch * blocks, device="cuda", generator=gen).to(torch.int32).view(batch, blocks)
    return table, batch * blocks, page


def to_pool(rows, table, pages, page, fill=0):
    """rows [B, capacity, ...] laid out as a page pool."""
    batch, capacity = rows.shape[:2]
    pool = torch.full((pages, page) + rows.shape[2:], fill, dtype=torch.float32, device="cuda").to(rows.dtype) \
        if rows.dtype not in (torch.uint8, torch.float8_e4m3fn) else torch.zeros((pages, page) + rows.shape[2:], dtype=torch.uint8, device="cuda")
    data = rows.view(torch.uint8) if rows.dtype == torch.float8_e4m3fn else rows
    for b in range(batch):
        for t0 in range(0, capacity, page):
            p = int(table[b, t0 // page]) if table is not None else b
            n = min(page, capacity - t0)
            pool[p, :n] = data[b, t0:t0 + n]
    return pool.view(torch.float8_e4m3fn) if rows.dtype == torch.float8_e4m3fn else pool


# ---- the 8-bit cache -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,tokens,heads,dim,page", [
    (1, 1, 1, 64, 0), (3, 5, 2, 128, 16), (2, 33, 4, 256, 7), (2, 9, 3, 72, 16), (2, 4, 2, 1, 0), (1, 6, 2, 7, 5), (5, 2, 12, 64, 64),
    (2, 3, 1, 200, 1)])
def test_kv8_rows(dtype, batch, tokens, heads, dim, page):
    gen, rnd = random(tokens * dim)
    start = torch.tensor([3 * b for b in range(batch)], **INT)
    capacity = 3 * batch + tokens
    table, pages, size = pages_of(batch, capacity, page, gen)
    k_pool, v_pool = (torch.full((pages, size, heads, dim), 0x55, dtype=torch.uint8, device="cuda") for _ in range(2))
    k_s, v_s = (torch.full((pages, size, heads), 0x77, dtype=torch.uint8, device="cuda") for _ in range(2))
    x = (rnd(batch, tokens, heads, dim) * 2.0 ** torch.randint(-30, 30, (batch, tokens, heads, 1), device="cuda", generator=gen)).to(dtype)
    y = rnd(batch, tokens, heads, 2, dim).to(dtype)[..., 1, :]   # strided rows
    x.view(-1)[0] = 448.0 * 2.0 ** 3
    y[0, 0, 0] = 0.0
    pools = k_pool.view(torch.float8_e4m3fn), v_pool.view(torch.float8_e4m3fn), k_s, v_s
    kv8_append(x, y, *pools, start, block_table=table)
    got = kv8_read(*pools, start, tokens, block_table=table, dtype=torch.float32)
    for value, rows in zip(got, (x, y)):
        held, _ = e8m0_rows(rows)
        assert torch.equal(value.double(), held)
    for value, exact in zip(kv8_read(*pools, start, tokens, block_table=table), got):
        assert torch.equal(value.float(), exact)   # every value held is exact in bf16
    # what the cache holds is held again as it is (a largest value that was rounded down to 448 * 2^(n - 1) takes the next
    # smaller scale, at which the row's codes stand for the same values: E4M3 values times two are E4M3 values, or
    # above 448, and none is); the slots around the rows keep what they had
    kv8_append(*got, *pools, start, block_table=table)
    for value, first in zip(kv8_read(*pools, start, tokens, block_table=table, dtype=torch.float32), got):
        assert torch.equal(value, first)
    written = torch.zeros(pages, size, dtype=torch.bool, device="cuda")
    for b in range(batch):
        for t in range(3 * b, 3 * b + tokens):
            written[int(table[b, t // size]) if page else b, t % size] = True
    assert (k_pool[~written] == 0x55).all() and (v_s[~written] == 0x77).all()
    assert _capi.kernel_status() == 0


def test_kv8_extremes():
    """The largest magnitudes, the smallest, the border between two scales, infinities and NaN."""
    top, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    rows = [[0.0, -0.0], [tiny, 0.0], [2.0 ** -126, -tiny], [448.0, 17.0], [448.0001, 17.0], [449.0, -448.0], [top, -top], [top, 1.0],
            [1.0, 2.0 ** -9], [1.75, 2.0 ** -18], [1.0, 17.0 / 16], [1.0, 19.0 / 16], [math.inf, 1.0], [-math.inf, 0.0], [math.nan, 1.0],
            [2.0 ** -118 * 448, 1e-40], [2.0 ** -127 * 448, 2.0 ** -136], [2.0 ** -127 * 449, 2.0 ** -136]]
    for dim in (8, 2):
        x = torch.tensor(rows, device="cuda").repeat(1, dim // 2).view(1, len(rows), 1, dim)
        pools = [torch.zeros(1, len(rows), 1, dim, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
        pools += [torch.zeros(1, len(rows), 1, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(x, -x, *pools, torch.zeros(1, **INT))
        for sign, value in zip((1, -1), kv8_read(*pools, torch.zeros(1, **INT), len(rows), dtype=torch.float32)):
            held, scale = e8m0_rows(sign * x)
            assert torch.equal(value.double().nan_to_num(nan=7.5), held.nan_to_num(nan=7.5))
            assert torch.equal(pools[2], scale)
    assert _capi.kernel_status() == 0


def test_kv8_counts_and_bad_slots():
    """Tokens behind counts[b] are neither written nor read; slots outside the pages, and pages outside the pool,
    are reported and left out."""
    gen, rnd = random(1)
    x = rnd(3, 4, 2, 64).bfloat16()
    new = lambda: [torch.zeros(3, 8, 2, 64, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)] + [  # noqa: E731
        torch.zeros(3, 8, 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    pools, counts = new(), torch.tensor([4, 0, 2], **INT)
    kv8_append(x, x, *pools, None, counts=counts)
    k, _ = kv8_read(*pools, torch.zeros(3, **INT), 4, counts=counts)
    whole, _ = e8m0_rows(x)
    for b, n in enumerate((4, 0, 2)):
        assert torch.equal(k[b, :n].double(), whole[b, :n]) and not k[b, n:].any()
        assert not pools[0].view(torch.uint8)[b, n:].any()
    assert _capi.kernel_status() == 0
    # sequence 1 runs past its page, sequence 2 starts before it
    pools = new()
    kv8_append(x, x, *pools, torch.tensor([0, 6, -3], **INT))
    assert _capi.kernel_status() & 0xff == 2
    codes = pools[0].view(torch.uint8)
    assert codes[0, :4].any(-1).all() and codes[1, 6:].any(-1).all() and not codes[1, :6].any() and codes[2, 0].any(-1).all()
    assert not codes[2, 1:].any()
    pools = new()
    table = torch.tensor([[2], [3], [-1]], **INT)
    kv8_append(x, x, *pools, None, block_table=table)
    assert _capi.kernel_status() & 0xff == 3
    codes = pools[0].view(torch.uint8)
    assert codes[2, :4].any(-1).all() and not codes[:2].any()


@pytest.mark.parametrize("store", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("batch,nodes,heads,dim,page", [(1, 1, 1, 64, 0), (4, 13, 2, 128, 16), (3, 128, 4, 256, 7), (2, 9, 3, 5, 4), (3, 31, 1, 6, 0)])
def test_keep_moves_the_path(store, batch, nodes, heads, dim, page):
    gen, _ = random(nodes + dim)
    capacity = 20 + nodes
    table, pages, size = pages_of(batch, capacity, page, gen)
    raw = lambda *s: torch.randint(0, 255, s, dtype=torch.uint8, device="cuda", generator=gen)  # noqa: E731
    element = torch.empty((), dtype=store).element_size()
    pools = [raw(pages, size, heads, dim * element).view(store) for _ in range(2)]
    scales = [raw(pages, size, heads) for _ in range(2)] if element == 1 else [None, None]
    prefix = torch.randint(0, 20, (batch,), device="cuda", generator=gen).int()
    accepted = torch.randint(0, nodes + 1, (batch,), device="cuda", generator=gen).int()
    accepted[0] = nodes if nodes > 20 else min(nodes, 3)
    path = torch.full((batch, nodes), -1, **INT)
    for b in range(batch):
        n = int(accepted[b])
        path[b, :n] = torch.randperm(nodes, device="cuda", generator=gen)[:n].sort().values.int()
    where = lambda b, t: (int(table[b, t // size]) if page else b, t % size)  # noqa: E731
    want = [t.clone() if t is not None else None for t in pools + scales]
    for b in range(batch):
        for i in range(int(accepted[b])):
            for t, w in zip(pools + scales, want):
                if t is not None:
                    w[where(b, int(prefix[b]) + i)] = t[where(b, int(prefix[b]) + int(path[b, i]))]
    kv_keep(*pools, prefix, path, accepted, block_table=table, k_scales=scales[0], v_scales=scales[1])
    for t, w in zip(pools + scales, want):
        if t is not None:
            assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))
    assert _capi.kernel_status() == 0


def test_keep_leaves_a_bad_path_alone():
    for path, accepted in (([0, 2, 2], 3), ([1, 0, 2], 2), ([0, 1, 3], 3), ([-1, 1, 2], 1), ([0, 1, 2], 4), ([0, 1, 2], -1)):
        pool = torch.arange(8 * 64, device="cuda").float().view(1, 8, 1, 64)
        other = pool.clone()
        kv_keep(pool, other, torch.ones(1, **INT), torch.tensor([path], **INT), torch.tensor([accepted], **INT))
        assert _capi.kernel_status() & 0xff == 5
        assert torch.equal(pool, other) and torch.equal(pool.view(-1), torch.arange(8 * 64, device="cuda").float())


# ---- attention of a tree of drafts -----------------------------------------------------------------------------
def random_parents(batch, nodes, gen):
    return (torch.rand(batch, nodes, device="cuda", generator=gen) * torch.arange(1, nodes + 1, device="cuda")).int() - 1


def attention_case(store, batch, nodes, hq, hkv, dim, longest, page, *, tree, ragged=True, gate=False, seed=0, dtype=torch.bfloat16,
                   out_dtype=None, rounded=False, lengths=None, share=1):
    """Runs gqa_tree_decode on a pool whose unused slots hold NaN, and holds it to the 64-bit model."""
    gen, rnd = random(seed + nodes * 131 + longest)
    capacity = longest + nodes
    table, pages, size = pages_of(batch, capacity, page, gen)
    prefix = torch.randint(0, longest + 1, (batch,), device="cuda", generator=gen).int() if lengths is None else torch.tensor(lengths, **INT)
    if lengths is None:
        prefix[0] = longest
    counts = torch.randint(0, nodes + 1, (batch,), device="cuda", generator=gen).int() if ragged else None
    if ragged:
        counts[0] = nodes
    parents = random_parents(batch, nodes, gen) if tree else None
    k, v = (rnd(batch, capacity, hkv, dim) for _ in range(2))
    scales = [None, None]
    if store == torch.float8_e4m3fn:
        rows = [torch.zeros(batch, capacity, hkv, dim, dtype=store, device="cuda") for _ in range(2)]
        rows += [torch.zeros(batch, capacity, hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k, v, *rows)
        k, v = kv8_read(*rows, torch.zeros(batch, **INT), capacity, dtype=torch.float32)
    else:
        rows = [k.to(store), v.to(store)]
        k, v = (r.float() for r in rows)
    used = torch.arange(capacity, device="cuda")[None] < (prefix + (counts if ragged else nodes))[:, None]
    for r in rows[:2]:
        if r.element_size() == 1:
            r.view(torch.uint8)[~used] = 0x7f
        else:
            r[~used] = math.nan
    for r in rows[2:]:
        r[~used] = 255
    laid = [to_pool(r, table, pages, size) for r in rows]
    scales = laid[2:] or [None, None]
    q = rnd(batch, nodes, hq, dim).to(dtype)
    g = rnd(batch, nodes, hq, 2, dim).to(dtype)[:, :, :, 1] if gate else None
    out = torch.full((batch, nodes, hq, dim), 7.5, dtype=out_dtype or dtype, device="cuda")
    call = lambda o: gqa_tree_decode(q, laid[0], laid[1], prefix, longest, parents=parents, counts=counts, block_table=table,  # noqa: E731
                                     k_scales=scales[0], v_scales=scales[1], gate=g, round_to_bfloat16=rounded, out=o, want_lse=True)
    got, lse = call(out)
    again, lse_again = call(torch.full_like(out, 7.5))
    assert torch.equal(got, again) and torch.equal(lse, lse_again)   # one order of summation
    for b in range(batch):
        n, length = int(counts[b]) if ragged else nodes, int(prefix[b])
        assert (got[b, n:] == 7.5).all()
        if n == 0:
            continue
        up = parents[b].tolist() if tree else list(range(-1, n - 1))
        want, mean, want_lse = tree_attention(q[b, :n].double(), k[b, :length + n].double(), v[b, :length + n].double(), length, up)
        # fp32 sums of `dim` products and of the keys' weights: 2^-20 of the mean magnitude.  On the tensor cores
        # each weight is rounded to bf16 (2^-8 of itself); the result's own rounding is 2^-8 of it.
        tensor_cores = dtype == torch.bfloat16 and got.dtype == torch.bfloat16 and store != torch.float32 and dim in (64, 128, 256)
        slack = mean * (2.0 ** -8 if tensor_cores else 2.0 ** -20)
        steps = 1 if got.dtype == torch.bfloat16 or rounded else 0
        if gate:
            factor = torch.sigmoid(g[b, :n].double())
            if rounded:
                factor, steps = factor.bfloat16().double(), 4   # core, factor (the same but at a tie), product
            want, slack = want * factor, slack * factor
        bound = slack * (1 + steps * 2.0 ** -8) + steps * 2.0 ** -8 * want.abs() * 1.01 + 1e-30
        off = (got[b, :n].double() - want).abs()
        assert (off <= bound).all(), (b, (off / bound).max().item())
        assert (lse[b, :n].double() - want_lse).abs().max().item() < 2e-5
    assert _capi.kernel_status() == 0


EIGHT, BF16, FP32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


@pytest.mark.parametrize("store", [EIGHT, BF16])
@pytest.mark.parametrize("batch,nodes,hq,hkv,dim,longest,page", [
    (1, 1, 24, 4, 256, 0, 0), (1, 1, 24, 4, 256, 63, 0), (3, 1, 24, 4, 256, 777, 16), (2, 13, 24, 4, 256, 130, 64), (1, 64, 24, 4, 256, 500, 0),
    (2, 128, 12, 2, 256, 70, 16), (1, 1, 40, 8, 128, 64, 0), (5, 1, 40, 8, 128, 2000, 16), (3, 5, 40, 8, 128, 65, 7), (2, 61, 40, 8, 128, 1000, 64),
    (1, 128, 10, 2, 128, 333, 48), (2, 26, 5, 1, 128, 200, 0), (4, 1, 12, 12, 64, 100, 16), (3, 8, 12, 12, 64, 1023, 1), (2, 127, 16, 1, 64, 129, 0),
    (40, 3, 12, 12, 64, 40, 16), (70, 1, 5, 1, 128, 300, 64),
    # few rows per KV head, either side of 8 and 16
    (3, 3, 40, 8, 128, 500, 16), (2, 8, 8, 8, 128, 129, 0), (2, 9, 4, 4, 128, 1000, 5), (2, 16, 12, 12, 64, 333, 16), (2, 17, 12, 12, 64, 333, 16),
    (3, 16, 2, 2, 128, 15, 0), (9, 8, 4, 4, 256, 700, 16), (2, 9, 4, 4, 256, 700, 16), (300, 2, 4, 2, 64, 90, 16), (1, 1, 8, 1, 128, 9000, 64)])
def test_tree_attention(store, batch, nodes, hq, hkv, dim, longest, page):
    attention_case(store, batch, nodes, hq, hkv, dim, longest, page, tree=nodes > 1)


@pytest.mark.parametrize("store", [EIGHT, BF16])
@pytest.mark.parametrize("nodes,hq,hkv,dim,longest", [(1, 24, 4, 256, 200), (7, 24, 4, 256, 64), (33, 40, 8, 128, 191), (60, 12, 12, 64, 5)])
@pytest.mark.parametrize("rounded", [False, True])
def test_gate_chain_and_prefixes_at_the_tile_borders(store, nodes, hq, hkv, dim, longest, rounded):
    lengths = [longest, 0, 1, max(0, longest - nodes), longest // 2, min(longest, 64 - nodes % 64)]
    attention_case(store, 6, nodes, hq, hkv, dim, longest, 16, tree=False, gate=True, rounded=rounded, lengths=lengths)


@pytest.mark.parametrize("store,dtype,out_dtype,dim,hq,hkv", [
    (FP32, FP32, FP32, 128, 4, 2), (FP32, BF16, BF16, 64, 4, 4), (BF16, FP32, FP32, 256, 6, 1), (BF16, BF16, FP32, 128, 5, 1), (EIGHT, FP32, FP32, 128, 4, 2),
    (EIGHT, FP32, BF16, 64, 4, 2), (BF16, BF16, BF16, 72, 4, 2), (EIGHT, BF16, BF16, 33, 3, 1), (FP32, FP32, FP32, 1, 2, 1), (EIGHT, BF16, FP32, 7, 2, 2)])
def test_other_types_and_widths(store, dtype, out_dtype, dim, hq, hkv):
    for nodes, longest in ((1, 0), (6, 37), (17, 300)):
        attention_case(store, 3, nodes, hq, hkv, dim, longest, 5, tree=True, dtype=dtype, out_dtype=out_dtype)


def test_one_node_is_gqa_decode():
    gen, rnd = random(5)
    k, v = rnd(4, 500, 8, 128).bfloat16(), rnd(4, 500, 8, 128).bfloat16()
    q, lens = rnd(4, 40, 128).bfloat16(), torch.tensor([1, 64, 333, 500], **INT)
    plain, plain_lse = gqa_decode(q, k, v, lens, 500, want_lse=True)
    got, lse = gqa_tree_decode(q[:, None], k, v, lens - 1, 499, want_lse=True)
    # bf16 weights (2^-8 of a mean of |v| below 1) and two roundings to bf16
    assert (got[:, 0].float() - plain.float()).abs().max().item() <= 2.0 ** -8 + 2.0 ** -7 * plain.float().abs().max().item()
    assert (lse[:, 0] - plain_lse).abs().max().item() < 2e-5


@pytest.mark.parametrize("store", [EIGHT, BF16, FP32])
@pytest.mark.parametrize("dim,hq,hkv", [(128, 10, 2), (256, 6, 1), (64, 4, 4), (128, 2, 2), (256, 1, 1), (64, 2, 1)])
def test_what_a_node_does_not_see_does_not_reach_it(store, dim, hq, hkv):
    """A row of infinities or NaN among the drafts (its keys, its values or both): nodes that see it get NaN, the
    others what they get without it."""
    gen, rnd = random(dim)
    prefix, parents = 70, torch.tensor([[-1, 0, 0, 1, -1, 4, 2, 3]], **INT)
    k, v = rnd(1, 80, hkv, dim), rnd(1, 80, hkv, dim)
    q = rnd(1, 8, hq, dim).bfloat16()
    at = torch.tensor([prefix], **INT)

    def run(k, v):
        if store != EIGHT:
            return gqa_tree_decode(q, k.to(store), v.to(store), at, prefix, parents=parents)
        rows = [torch.zeros(1, 80, hkv, dim, dtype=store, device="cuda") for _ in range(2)]
        rows += [torch.zeros(1, 80, hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k, v, *rows)
        return gqa_tree_decode(q, rows[0], rows[1], at, prefix, parents=parents, k_scales=rows[2], v_scales=rows[3])
    clean = run(k, v)
    assert torch.isfinite(clean).all()
    sees = [1, 3, 7]   # node 1 and its descendants
    for bad_k, bad_v in ((math.nan, None), (None, math.nan), (None, math.inf), (math.inf, -math.inf)):
        kk, vv = k.clone(), v.clone()
        if bad_k is not None:
            kk[0, prefix + 1] = bad_k
        if bad_v is not None:
            vv[0, prefix + 1] = bad_v
        got = run(kk, vv)
        for node in range(8):
            if node not in sees:
                assert torch.equal(got[0, node], clean[0, node]), (bad_k, bad_v, node)
            elif store == EIGHT or bad_k is not None and math.isnan(bad_k):
                assert torch.isnan(got[0, node]).all()
            else:
                assert not torch.isfinite(got[0, node]).any()
    assert _capi.kernel_status() == 0


def test_head_shard_of_a_wider_cache():
    """Two of eight KV heads, addressed in place by pointer and stride."""
    gen, rnd = random(9)
    k, v, q = rnd(2, 300, 8, 128).bfloat16(), rnd(2, 300, 8, 128).bfloat16(), rnd(2, 5, 10, 128).bfloat16()
    at = torch.tensor([290, 100], **INT)
    whole = gqa_tree_decode(q, k[:, :, 4:6].contiguous(), v[:, :, 4:6].contiguous(), at, 290)
    assert torch.equal(gqa_tree_decode(q, k[:, :, 4:6], v[:, :, 4:6], at, 290), whole)


def test_bad_lengths_pages_and_parents_are_reported():
    gen, rnd = random(3)
    k, v, q = rnd(2, 64, 2, 128).bfloat16(), rnd(2, 64, 2, 128).bfloat16(), rnd(2, 4, 4, 128).bfloat16()
    at = torch.tensor([10, 20], **INT)
    good = gqa_tree_decode(q, k, v, at, 60)
    for prefix, kind in (([10, -4], 2), ([10, 61], 2)):
        out = gqa_tree_decode(q, k, v, torch.tensor(prefix, **INT), 60)
        assert _capi.kernel_status() & 0xff == kind and torch.equal(out[0], good[0])
    out = gqa_tree_decode(q, k, v, at, 60, counts=torch.tensor([4, 9], **INT))
    assert _capi.kernel_status() & 0xff == 2 and torch.equal(out, good)
    parents = torch.tensor([[-1, 0, 1, 2], [-1, 0, 7, -9]], **INT)
    out = gqa_tree_decode(q, k, v, at, 60, parents=parents)
    assert _capi.kernel_status() & 0xff == 5 and torch.equal(out[0], good[0])
    parents[1, 2:] = -1   # what such parents are taken for
    assert torch.equal(out, gqa_tree_decode(q, k, v, at, 60, parents=parents))
    table = torch.tensor([[0, 1], [2, 99]], **INT)
    pools = k.view(4, 32, 2, 128), v.view(4, 32, 2, 128)
    out = gqa_tree_decode(q, *pools, at, 60, block_table=table)
    assert torch.equal(out, good) and _capi.kernel_status() == 0   # the bad page holds no slot in use
    out = gqa_tree_decode(q, *pools, torch.tensor([10, 40], **INT), 60, block_table=table)
    assert _capi.kernel_status() & 0xff == 3 and torch.equal(out[0], good[0]) and torch.isfinite(out).all()


def test_other_streams_graphs_and_workspaces():
    """Two captured graphs of different sizes, replayed at the same time on two streams, beside eager calls."""
    gen, rnd = random(11)
    make = lambda n, hq, hkv, d, t: (rnd(2, n, hq, d).bfloat16(), rnd(2, t, hkv, d).bfloat16(), rnd(2, t, hkv, d).bfloat16(),  # noqa: E731
                                     torch.tensor([t - n, t // 2], **INT), t - n)
    cases = [make(1, 40, 8, 128, 3000), make(30, 24, 4, 256, 1500)]
    want = [gqa_tree_decode(*c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(gqa_tree_decode(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = [gqa_tree_decode(*c) for c in reversed(cases)]
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
        for o, w in zip(eager, reversed(want)):
            assert torch.equal(o, w)
    with pytest.raises(PlutoStatusError, match="workspace"):
        gqa_tree_decode(*cases[0], workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))


# ---- the prepare step and the cached layers --------------------------------------------------------------------
def step_inputs(p, n, rnd, dtype=torch.bfloat16):
    return (rnd(n, p.query_heads, 2, p.head_dim).to(dtype), rnd(n, p.key_value_heads, p.head_dim).to(dtype),
            rnd(n, p.key_value_heads, p.head_dim).to(dtype))


@pytest.mark.parametrize("rounded", [True, False])
@pytest.mark.parametrize("hq,hkv,dim,rotary", [(24, 4, 256, 64), (40, 8, 128, 128), (4, 2, 36, 12)])
def test_draft_prepare_is_the_cached_steps_prepare(rounded, hq, hkv, dim, rotary):
    """Every node's rows are those that a step at its own position writes, bit for bit, in fp32 and bf16 caches;
    8-bit rows are the append of them."""
    gen, rnd = random(dim)
    dtype = torch.bfloat16 if rounded else torch.float32
    p = FullAttentionParameters(hq, hkv, dim, rotary, 60, round_to_bfloat16=rounded)
    q_norm, k_norm = rnd(dim) * 0.1, rnd(dim) * 0.1
    parents = torch.tensor([[-1, 0, 0, 2, -1, 4, 3]], **INT)
    depth, first = [0, 1, 1, 2, 0, 1, 3], 17
    qg, k, v = step_inputs(p, 7, rnd, dtype)
    caches = {store: KeyValueCache.Create(60, hkv, dim, dtype=store) for store in (FP32, BF16, EIGHT)}
    queries = {}
    for store, cache in caches.items():
        cache.position_ = first
        queries[store] = draft_prepare(qg[None, :, :, 0], k[None], v[None], q_norm, k_norm, cache.device_position(), **cache.pool(),
                                       rotary_dim=rotary, rms_norm_epsilon=p.rms_norm_epsilon, rope_theta=p.rope_theta,
                                       round_to_bfloat16=rounded, parents=parents)
        assert torch.equal(queries[store], queries[FP32])
    want_k, want_v = [], []
    for i in range(7):
        cache = KeyValueCache.Create(60, hkv, dim, dtype=FP32)
        cache.position_ = first + depth[i]
        CachedAttentionStep(p, cache, qg[i], k[i], v[i], q_norm, k_norm, torch.empty(hq, dim, dtype=dtype, device="cuda"))
        want_k.append(cache.keys()[first + depth[i]].clone())
        want_v.append(cache.values()[first + depth[i]].clone())
    want_k, want_v = torch.stack(want_k), torch.stack(want_v)
    assert torch.equal(caches[FP32].keys()[first:first + 7], want_k) and torch.equal(caches[FP32].values()[first:first + 7], want_v)
    assert torch.equal(caches[BF16].keys()[first:first + 7], want_k.bfloat16())
    eight = KeyValueCache.Create(60, hkv, dim, dtype=EIGHT)
    pool = eight.pool()
    kv8_append(want_k[None], want_v[None], **pool, positions=torch.tensor([first], **INT))
    got = caches[EIGHT].pool()
    for name in pool:
        assert torch.equal(pool[name].view(torch.uint8), got[name].view(torch.uint8)), name
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("hq,hkv,dim,rotary", [(24, 4, 256, 64), (40, 8, 128, 128), (4, 2, 36, 12)])
def test_cached_step_over_an_8_bit_cache(hq, hkv, dim, rotary):
    gen, rnd = random(dim + 1)
    p = FullAttentionParameters(hq, hkv, dim, rotary, 40)
    cache = KeyValueCache.Create(40, hkv, dim, dtype=EIGHT)
    q_norm, k_norm = rnd(dim) * 0.1, rnd(dim) * 0.1
    for t in range(20):
        qg, k, v = step_inputs(p, 1, rnd)
        out = torch.empty(hq, dim, dtype=BF16, device="cuda")
        CachedAttentionStep(p, cache, qg[0], k[0], v[0], q_norm, k_norm, out)
        assert cache.position() == t + 1
        scratch = KeyValueCache.Create(40, hkv, dim)
        query = draft_prepare(qg[None, :, :, 0], k[None], v[None], q_norm, k_norm, torch.tensor([t], **INT), **scratch.pool(), rotary_dim=rotary,
                              rms_norm_epsilon=p.rms_norm_epsilon, rope_theta=p.rope_theta)
        held = [x[0].double() for x in kv8_read(**cache.pool(), positions=torch.zeros(1, **INT), tokens=t + 1)]
        want, mean, _ = tree_attention(query[0].double(), held[0], held[1], t, [-1])
        factor = torch.sigmoid(qg[:, :, 1].double()).bfloat16().double()
        bound = factor * (mean * 2.0 ** -8 + 4 * 2.0 ** -8 * want.abs()) * 1.02 + 1e-30
        assert ((out.double() - want[0] * factor[0]).abs() <= bound[0]).all()
    with pytest.raises(PlutoStatusError, match="8-bit"):
        CachedAttentionStep(p, cache, qg[0], k[0], v[0], q_norm, k_norm, out, torch.empty(hq, 21, device="cuda"))
    assert cache.position() == 20
    for _ in range(20):
        CachedAttentionStep(p, cache, qg[0], k[0], v[0], q_norm, k_norm, out)
    with pytest.raises(PlutoStatusError, match="capacity"):
        CachedAttentionStep(p, cache, qg[0], k[0], v[0], q_norm, k_norm, out)
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("store", [EIGHT, BF16, FP32])
@pytest.mark.parametrize("hq,hkv,dim,rotary", [(24, 4, 256, 64), (10, 2, 128, 128)])
@pytest.mark.parametrize("strict", [0.2, 0.0])   # (at 0 the first child of every node is accepted)
def test_a_speculative_step_is_the_steps_of_its_accepted_path(store, hq, hkv, dim, rotary, strict):
    """Drafts, attention, verification and the cache step together: three rounds of a tree of 16 nodes.  What the
    cache holds behind each round is, bit for bit, what one step per accepted token leaves, and the
    accepted nodes' outputs are those steps' within two bf16 results of one attention."""
    gen, rnd = random(dim + 2)
    p = FullAttentionParameters(hq, hkv, dim, rotary, 100)
    q_norm, k_norm = rnd(dim) * 0.1, rnd(dim) * 0.1
    drafted, stepped = (KeyValueCache.Create(100, hkv, dim, dtype=store) for _ in range(2))
    vocab, nodes, total = 50, 16, 0
    head = rnd(hq * dim, vocab) / 4
    for step in range(3):
        parents = random_parents(1, nodes, gen)
        qg, k, v = step_inputs(p, nodes, rnd)
        out = torch.empty(nodes, hq, dim, dtype=BF16, device="cuda")
        CachedDraftStep(p, drafted, qg, k, v, q_norm, k_norm, out, parents[0])
        assert drafted.position() == total
        logits = torch.cat([torch.zeros(1, vocab, device="cuda"), out.reshape(nodes, -1).float() @ head])
        target = torch.softmax(logits, -1)[None]
        # the drafts are the target's likeliest tokens after their parents, so that some are accepted
        likely = target[0].topk(4).indices
        tokens = torch.stack([likely[int(parents[0, i]) + 1, i % 4] for i in range(nodes)])[None].int()
        u, u_last = torch.rand(1, nodes, device="cuda", generator=gen) * strict, torch.rand(1, device="cuda", generator=gen)
        verdict = verify_drafts(target, tokens, u, u_last, parents=parents)
        want = verify(target[0].tolist(), tokens[0].tolist(), u[0].tolist(), float(u_last), parents[0].tolist(), nodes)
        assert (int(verdict.accepted), verdict.path[0].tolist(), verdict.tokens[0].tolist()) == want
        count = drafted.Keep(verdict.path[0], verdict.accepted)
        assert count == want[0] and drafted.position() == total + count
        total += count
        for i in want[1][:count]:
            one = torch.empty(hq, dim, dtype=BF16, device="cuda")
            CachedAttentionStep(p, stepped, qg[i], k[i], v[i], q_norm, k_norm, one)
            assert (one.float() - out[i].float()).abs().max().item() <= 2.0 ** -6 * max(1.0, one.float().abs().max().item())
        for name, pool in drafted.pool().items():
            if pool is not None:
                assert torch.equal(pool.view(torch.uint8)[0, :total], stepped.pool()[name].view(torch.uint8)[0, :total]), name
    assert (total > 0 or strict) and _capi.kernel_status() == 0
    with pytest.raises(PlutoStatusError, match="capacity"):
        full = KeyValueCache.Create(100, hkv, dim, dtype=store)
        full.position_ = 90
        CachedDraftStep(p, full, qg, k, v, q_norm, k_norm, out, parents[0])
    with pytest.raises(PlutoStatusError, match="do not match"):
        CachedDraftStep(p, drafted, qg, k[:3], v, q_norm, k_norm, out, parents[0])


# ---- verification ----------------------------------------------------------------------------------------------
def verify_case(seed, batch, nodes, vocab, form, dtype=torch.float32, counts=True, dyadic=False, zeros=0.3):
    gen, _ = random(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)  # noqa: E731
    if dyadic:   # products and sums are exact whatever the precision, and ties happen
        row = lambda n: torch.randint(0, 3, (batch, n, vocab), device="cuda", generator=gen) / 2.0 ** 6  # noqa: E731
        u, u_last = (torch.randint(0, 8, s, device="cuda", generator=gen) / 8.0 for s in ((batch, nodes), (batch,)))
    else:
        def row(n):
            x = rand(batch, n, vocab) ** 4 * (rand(batch, n, vocab) > zeros)
            return x / x.sum(-1, keepdim=True).clamp(min=1e-9)
        u, u_last = rand(batch, nodes) * rand(batch, 1), rand(batch)
    p, q = row(nodes + 1).to(dtype), row(nodes).to(dtype) if form == "drawn" else None
    parents = random_parents(batch, nodes, gen) if form == "tree" else None
    best = p[:, :nodes].float().argmax(-1)
    tokens = torch.where(rand(batch, nodes) < 0.5, best, torch.randint(0, min(vocab, 6), (batch, nodes), device="cuda", generator=gen)).int()
    n = torch.randint(0, nodes + 1, (batch,), device="cuda", generator=gen).int() if counts else None
    return p, tokens, u.float(), u_last.float(), parents, n, q


def check_verify(p, tokens, u, u_last, parents, counts, q):
    got = verify_drafts(p, tokens, u, u_last, parents=parents, counts=counts, draft_probs=q)
    batch, nodes = tokens.shape
    host = lambda t: None if t is None else t.double().tolist() if t.is_floating_point() else t.tolist()  # noqa: E731
    p, q, tokens, u, u_last, parents, counts = (host(t) for t in (p, q, tokens, u, u_last, parents, counts))
    result = [t.tolist() for t in got]
    for b in range(batch):
        want = verify(p[b], tokens[b], u[b], u_last[b], parents[b] if parents else None, counts[b] if counts else nodes, q[b] if q else None)
        assert (result[0][b], result[1][b], result[2][b]) == want, b
    return result


@pytest.mark.parametrize("form", ["drawn", "given", "tree"])
@pytest.mark.parametrize("batch,nodes,vocab", [(40, 1, 1), (40, 3, 2), (60, 8, 5), (30, 17, 33), (10, 31, 1000), (6, 128, 129), (3, 5, 4097), (2, 7, 50257)])
def test_verify(form, batch, nodes, vocab):
    check_verify(*verify_case(nodes, batch, nodes, vocab, form))
    check_verify(*verify_case(nodes + 1, batch, nodes, vocab, form, dyadic=True))
    check_verify(*verify_case(nodes + 2, batch, nodes, vocab, form, dtype=torch.bfloat16, counts=False))
    assert _capi.kernel_status() == 0


def test_verify_edges():
    p, tokens, u, u_last, parents, counts, _ = verify_case(1, 12, 6, 40, "tree", counts=False)
    u[0], u_last[0] = 0.0, 0.0
    u[1], u_last[1] = 1 - 2.0 ** -24, 1 - 2.0 ** -24
    p[2] = 0.0                                    # nothing to draw from
    p[3, :, 7] = math.nan
    p[4, :, 3] = math.inf
    p[5] = 0.0
    p[5, :, 39] = 1.0                             # all in the last token
    p[6] = 0.0
    p[6, :, 0] = 2.0 ** -140                      # a subnormal sum
    tokens[7] = 3                                 # the same token everywhere
    result = check_verify(p, tokens, u, u_last, parents, counts, None)
    assert result[2][2][result[0][2]] == -1
    assert _capi.kernel_status() == 0
    # a star: 128 children of the last cached token
    p, tokens, u, u_last, _, _, _ = verify_case(2, 4, 128, 300, "given", counts=False)
    tokens[:] = torch.randint(0, 300, tokens.shape, device="cuda").int()
    check_verify(p, tokens, u + 0.9, u_last, torch.full((4, 128), -1, **INT), None, None)
    # p == q: nothing is left after a refusal, which u * q < p makes only at u = 1 - 2^-24 and above; the row itself then
    p, tokens, u, u_last, _, _, q = verify_case(3, 4, 3, 64, "drawn", counts=False)
    p[:, 0], q[:, 0] = 0.0, 1.0 / 64
    check_verify(p, tokens, u, u_last, None, None, q)
    # tokens and parents out of range are reported and refused
    for bad in (-1, 40, 2 ** 30):
        p, tokens, u, u_last, parents, _, _ = verify_case(4, 3, 5, 40, "tree", counts=False)
        tokens[1, 2] = bad
        check_verify(p, tokens, u, u_last, parents, None, None)
        assert _capi.kernel_status() & 0xff == 5
    p, tokens, u, u_last, parents, _, _ = verify_case(5, 3, 5, 40, "tree", counts=False)
    parents[0, 1], parents[2, 3] = 1, -7
    check_verify(p, tokens, u, u_last, parents, None, None)
    assert _capi.kernel_status() & 0xff == 5
    verify_drafts(p, tokens, u, u_last, counts=torch.tensor([6, -1, 2], **INT))
    assert _capi.kernel_status() & 0xff == 2


def test_verify_vocabulary_limit_and_last_chunks():
    """Every chunk border of a large row can hold the drawn token."""
    vocab = 1048576
    p = torch.zeros(1, 2, vocab, device="cuda")
    spots = [0, 31, 32, 8191, 8192, 131071, 131072, 524287, vocab - 1]
    p[:, :, spots] = 1.0 / len(spots)
    for i, x in enumerate(spots):
        got = verify_drafts(p, torch.tensor([[5]], **INT), torch.tensor([[0.5]], device="cuda"),
                            torch.tensor([(i + 0.5) / len(spots)], device="cuda"))
        assert got.tokens.tolist() == [[x, -1]] and got.accepted.tolist() == [0]


@pytest.mark.parametrize("refused", [
    lambda: kv8_append(torch.zeros(1, 1, 1, 64, device="cuda"), torch.zeros(1, 1, 1, 64, device="cuda"),
                       *[torch.zeros(1, 4, 1, 64, dtype=BF16, device="cuda")] * 2, None, None),
    lambda: gqa_tree_decode(torch.zeros(2, 1, 4, 64, device="cuda", dtype=BF16), *[torch.zeros(1, 4, 2, 64, dtype=BF16, device="cuda")] * 2,
                            torch.zeros(2, **INT), 3),
    lambda: gqa_tree_decode(torch.zeros(1, 1, 4, 64, device="cuda", dtype=BF16), *[torch.zeros(1, 4, 2, 64, dtype=BF16, device="cuda")] * 2,
                            torch.zeros(1, dtype=torch.int64, device="cuda"), 3),
    lambda: gqa_tree_decode(torch.zeros(1, 1, 4, 64, device="cuda", dtype=BF16), *[torch.zeros(1, 4, 2, 64, dtype=BF16, device="cuda")] * 2,
                            torch.zeros(1, dtype=torch.int32), 3),
    lambda: gqa_tree_decode(torch.zeros(1, 1, 4, 64, device="cuda", dtype=BF16), *[torch.zeros(1, 4, 2, 64, dtype=EIGHT, device="cuda")] * 2,
                            torch.zeros(1, **INT), 3),
    lambda: gqa_tree_decode(torch.zeros(1, 1, 4, 64, device="cuda", dtype=BF16), *[torch.zeros(1, 4, 2, 64, dtype=BF16)] * 2,
                            torch.zeros(1, **INT), 3),
    lambda: gqa_tree_decode(torch.zeros(1, 1, 4, 32, device="cuda", dtype=BF16), *[torch.zeros(1, 4, 2, 64, dtype=BF16, device="cuda")] * 2,
                            torch.zeros(1, **INT), 3),
    lambda: verify_drafts(torch.zeros(1, 2, 9, device="cuda"), torch.zeros(1, 2, **INT), torch.zeros(1, 2, device="cuda"), torch.zeros(1, device="cuda")),
    lambda: verify_drafts(torch.zeros(1, 3, 9, device="cuda"), torch.zeros(1, 2, **INT), torch.zeros(1, 2, device="cuda"), torch.zeros(1, device="cuda"),
                          parents=torch.zeros(1, 2, **INT), draft_probs=torch.zeros(1, 2, 9, device="cuda")),
])
def test_refusals(refused):
    with pytest.raises(PlutoStatusError):
        refused()
