"""Attention of drafted tokens over 8-bit caches whose value rows have scales far from one, far from each other, or large
where a node does not see them."""
import math

import pytest
import torch

from drafts_double import seen_by, tree_attention
from pluto_b200 import _capi
from pluto_b200.layers import gqa_tree_decode

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")
EIGHT = torch.float8_e4m3fn
# (nodes, query heads, KV heads, width): up to 8 and 16 rows per KV head, up to 128, more than 128
SHAPES = [(1, 10, 2, 128), (3, 4, 4, 64), (1, 6, 1, 256), (3, 10, 2, 128), (20, 10, 2, 128), (30, 4, 4, 64), (20, 6, 1, 256), (40, 20, 4, 128), (70, 6, 3, 64)]


def values(codes, scales):
    """The float64 values of 8-bit rows."""
    power = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64, device="cuda"), scales.int() - 127)
    return codes.double() * power[..., None]


def hold_to_the_model(q, k, v, k_scales, v_scales, prefix, parents, at_least=0.5):
    """One sequence against the 64-bit model.  A weight is taken to fp16 times its row's 2^n relative to the largest 2^n that the
    node sees: off by 2^-11 of itself, and by 2^-25 of that largest 2^n where it is subnormal, against a sum of weights
    of 1 or more.  Scores and sums are in fp32 (2^-20 of a mean of |v|); the result is rounded once, to bf16."""
    nodes, hq, hkv = q.shape[1], q.shape[2], k.shape[2]
    up = parents[0].tolist()
    got, lse = gqa_tree_decode(q, k, v, torch.tensor([prefix], **INT), prefix, parents=parents, k_scales=k_scales, v_scales=v_scales,
                               round_to_bfloat16=False, want_lse=True)
    rows = slice(0, prefix + nodes)
    want, mean, want_lse = tree_attention(q[0].double(), values(k, k_scales)[0, rows], values(v, v_scales)[0, rows], prefix, up)
    seen = torch.cat([torch.ones(nodes, prefix, dtype=torch.bool), seen_by(up, nodes)], 1).cuda()
    n = v_scales[0, rows].double() - 127
    largest = torch.where(seen[:, :, None], n[None], -math.inf).amax(1)                     # [nodes, hkv]
    codes = torch.einsum("nt,thd->nhd", seen.double(), v[0, rows].double().abs())
    lost = (2.0 ** (largest - 25)[..., None] * codes).repeat_interleave(hq // hkv, 1)
    bound = mean * (2.0 ** -11 * 1.01 + 2.0 ** -20) + lost + 2.0 ** -8 * want.abs() * 1.01
    off = (got[0].double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    assert (bound < want.abs()).double().mean().item() > at_least                           # zeros would not pass
    assert (lse[0].double() - want_lse).abs().max().item() < 2e-5 * max(1.0, want_lse.abs().max().item())
    assert _capi.kernel_status() == 0
    return got


def case(nodes, hq, hkv, dim, prefix, powers, seed, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    rows = prefix + nodes
    k, v = rnd(1, rows, hkv, dim).to(EIGHT), (rnd(1, rows, hkv, dim) * 16).to(EIGHT)
    n = torch.tensor(powers, device="cuda")[torch.randint(0, len(powers), (1, rows, hkv), device="cuda", generator=gen)]
    q = (rnd(1, nodes, hq, dim) * spread).bfloat16()
    parents = (torch.rand(1, nodes, device="cuda", generator=gen) * torch.arange(1, nodes + 1, device="cuda")).int() - 1
    return q, k, v, torch.full((1, rows, hkv), 127, dtype=torch.uint8, device="cuda"), (n + 127).to(torch.uint8), parents


@pytest.mark.parametrize("prefix", [0, 1, 30, 64, 100, 333])
@pytest.mark.parametrize("powers", [[-16], [-24], [-40], [-80], [12], [30], [-12]])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_scales_far_from_one(nodes, hq, hkv, dim, powers, prefix):
    q, k, v, ks, vs, parents = case(nodes, hq, hkv, dim, prefix, powers, nodes + prefix)
    hold_to_the_model(q, k, v, ks, vs, prefix, parents, at_least=0.9)


@pytest.mark.parametrize("zero", [0, 70, -1])
@pytest.mark.parametrize("power", [-30, -12, -7, 0, 20])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_a_row_of_zeros_among_others(nodes, hq, hkv, dim, power, zero):
    """Its scale byte is 0; the others keep the weights that they have beside ordinary rows."""
    q, k, v, ks, vs, parents = case(nodes, hq, hkv, dim, 150, [power], nodes)
    v.view(torch.uint8)[0, zero] = 0
    vs[0, zero] = 0
    hold_to_the_model(q, k, v, ks, vs, 150, parents, at_least=0.8)


@pytest.mark.parametrize("places", ["prefix", "first tile"])
@pytest.mark.parametrize("powers", [(-40, -20), (-13, -26), (0, -14), (-14, 0), (7, -8)])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_scales_that_change_along_the_keys(nodes, hq, hkv, dim, powers, places):
    q, k, v, ks, vs, parents = case(nodes, hq, hkv, dim, 333, [powers[0]], nodes)
    vs[0, 64 if places == "first tile" else 300:] = 127 + powers[1]
    hold_to_the_model(q, k, v, ks, vs, 333, parents)


@pytest.mark.parametrize("prefix", [0, 1, 30, 64, 100, 333])
@pytest.mark.parametrize("powers", [[-20, -18], [-90, -70], [-110, -118], [-15, -22], [30, 27], [0, 40], [-50, 60]])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_scales_that_differ_from_row_to_row(nodes, hq, hkv, dim, powers, prefix):
    q, k, v, ks, vs, parents = case(nodes, hq, hkv, dim, prefix, powers, nodes + prefix)
    hold_to_the_model(q, k, v, ks, vs, prefix, parents, at_least=0.3)


@pytest.mark.parametrize("prefix", [0, 3, 60, 62, 130, 1000])
@pytest.mark.parametrize("k_power,v_power", [(0, 30), (0, 80), (0, 119), (30, 0), (80, 40), (-40, 9), (0, -40)])
@pytest.mark.parametrize("hq,hkv,dim", [(10, 2, 128), (6, 1, 256), (4, 4, 64), (2, 2, 128), (1, 1, 256), (40, 2, 64), (40, 1, 128)])
def test_a_finite_row_that_a_node_does_not_see_does_not_reach_it(hq, hkv, dim, k_power, v_power, prefix):
    """A draft whose rows have other scales than all others: bit for bit what its neighbours get beside an ordinary one."""
    up = [-1, 0, 0, 1, -1, 4, 2, 3]
    q, k, v, ks, vs, _ = case(8, hq, hkv, dim, prefix, [-7], dim + prefix)
    parents = torch.tensor([up], **INT)
    clean = hold_to_the_model(q, k, v, ks, vs, prefix, parents, at_least=0.8)
    ks[0, prefix + 1], vs[0, prefix + 1] = 127 + k_power, 127 + v_power
    if k_power <= 0:
        got = hold_to_the_model(q, k, v, ks, vs, prefix, parents, at_least=0.0)
    else:   # (scores that fp32 holds to some units only: of no interest beside their neighbours)
        got = gqa_tree_decode(q, k, v, torch.tensor([prefix], **INT), prefix, parents=parents, k_scales=ks, v_scales=vs, round_to_bfloat16=False)
    for node in (0, 2, 4, 5, 6):
        assert torch.equal(got[0, node], clean[0, node]), node


@pytest.mark.parametrize("prefix", [10, 700, 2500])
@pytest.mark.parametrize("powers", [[119], [100], [119, 112], [118, -90], [60, -60]])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_the_largest_scales_keep_small_weights(nodes, hq, hkv, dim, powers, prefix):
    """Weights over six powers of e, which add up to more than the largest does."""
    q, k, v, ks, vs, parents = case(nodes, hq, hkv, dim, prefix, powers, nodes + prefix, spread=2.0)
    hold_to_the_model(q, k, v, ks, vs, prefix, parents, at_least=0.3)
