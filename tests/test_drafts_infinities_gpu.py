"""Infinities in rows that a node sees, over bf16 and fp32 caches: scores of -infinity, of +infinity, and nothing else."""
import math

import pytest
import torch

from drafts_double import tree_attention
from pluto_b200 import _capi
from pluto_b200.layers import gqa_tree_decode

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")
SHAPES = [(1, 10, 2, 128), (3, 4, 4, 64), (1, 6, 1, 256), (3, 10, 2, 128), (20, 10, 2, 128), (30, 4, 4, 64), (20, 6, 1, 256), (40, 20, 4, 128), (70, 6, 3, 64)]
STORES = [torch.bfloat16, torch.float32]


def case(nodes, hq, hkv, dim, rows):
    gen = torch.Generator(device="cuda").manual_seed(nodes + dim)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    k, v, q = rnd(1, rows, hkv, dim).bfloat16(), rnd(1, rows, hkv, dim).bfloat16(), rnd(1, nodes, hq, dim).bfloat16()
    q[..., 7] = torch.where(q[..., 7] == 0, torch.ones_like(q[..., 7]), q[..., 7])
    return k, v, q


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("infinity", [math.inf, -math.inf])
@pytest.mark.parametrize("token", [0, 70, 199])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_one_infinite_key_channel(store, infinity, token, nodes, hq, hkv, dim):
    """Queries of its sign get NaN; for the others the row has a weight of zero."""
    prefix = 200
    k, v, q = case(nodes, hq, hkv, dim, prefix + nodes)
    k[0, token, :, 7] = infinity
    got, lse = gqa_tree_decode(q, k.to(store), v.to(store), torch.tensor([prefix], **INT), prefix, round_to_bfloat16=False, want_lse=True)
    up = q[0, :, :, 7] * infinity > 0
    assert torch.isnan(got[0][up]).all() and up.any() and (~up).any()
    rest = [x for x in range(prefix + nodes) if x != token]
    want, mean, want_lse = tree_attention(q[0].double(), k[0, rest].double(), v[0, rest].double(), prefix - 1, list(range(-1, nodes - 1)))
    # weights rounded to bf16 or better (2^-8 of a mean of |v|), the result rounded once
    off, bound = (got[0].double() - want).abs(), mean * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -8 * 1.01 * want.abs() + 1e-30
    assert (off <= bound)[~up].all() and (lse[0].double() - want_lse).abs()[~up].max().item() < 2e-5
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("prefix", [0, 5, 130])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_nothing_but_scores_of_minus_infinity(store, prefix, nodes, hq, hkv, dim):
    """A query without a finite score gets zeros, and minus infinity as the logarithm of its sum."""
    k, v, q = case(nodes, hq, hkv, dim, prefix + nodes)
    k[0, :, :, 7] = -math.inf
    got, lse = gqa_tree_decode(q, k.to(store), v.to(store), torch.tensor([prefix], **INT), prefix, round_to_bfloat16=False, want_lse=True)
    up = q[0, :, :, 7] < 0
    assert torch.isnan(got[0][up]).all()
    assert not got[0][~up].any() and (lse[0][~up] == -math.inf).all()
    assert _capi.kernel_status() == 0


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("token", [0, 70, 199, 200])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_one_value_channel_that_is_not_finite(store, value, token, nodes, hq, hkv, dim):
    """It leaves nothing finite in that channel of the nodes that see it, and nothing unless drafts hold it in the others."""
    prefix = 200
    k, v, q = case(nodes, hq, hkv, dim, prefix + nodes)
    clean = gqa_tree_decode(q, k.to(store), v.to(store), torch.tensor([prefix], **INT), prefix, round_to_bfloat16=False)
    v[0, token, :, 5] = value
    got = gqa_tree_decode(q, k.to(store), v.to(store), torch.tensor([prefix], **INT), prefix, round_to_bfloat16=False)
    assert not torch.isfinite(got[..., 5]).any()
    if token < prefix:
        others = [c for c in range(dim) if c != 5]
        assert torch.equal(got[..., others], clean[..., others])
    assert _capi.kernel_status() == 0
