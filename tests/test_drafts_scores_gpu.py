"""Attention of drafted tokens where scores are too large for their differences to mean anything."""
import math

import pytest
import torch

from drafts_double import tree_attention
from pluto_b200 import _capi
from pluto_b200.layers import gqa_tree_decode, kv8_append, kv8_read

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")
EIGHT, BF16, FP32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32
SHAPES = [(1, 10, 2, 128), (3, 4, 4, 64), (1, 6, 1, 256), (3, 10, 2, 128), (20, 10, 2, 128), (30, 4, 4, 64), (20, 6, 1, 256), (40, 20, 4, 128), (70, 6, 3, 64)]


@pytest.mark.parametrize("store", [EIGHT, BF16, FP32])
@pytest.mark.parametrize("power", [20, 28, 32, 40, 80, 100])
@pytest.mark.parametrize("token", [0, 70, 199])
@pytest.mark.parametrize("nodes,hq,hkv,dim", SHAPES)
def test_one_key_row_of_a_large_scale(store, nodes, hq, hkv, dim, power, token):
    """Queries that it scores above all others get its value row, the others what they get without it."""
    gen = torch.Generator(device="cuda").manual_seed(nodes + power)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    prefix, rows = 200, 200 + nodes
    k, v, q = rnd(1, rows, hkv, dim), rnd(1, rows, hkv, dim), rnd(1, nodes, hq, dim).bfloat16()
    k[0, token] = torch.where(k[0, token] < 0, -2.0 ** power, 2.0 ** power)
    scales = [None, None]
    if store == EIGHT:
        pools = [torch.zeros(1, rows, hkv, dim, dtype=store, device="cuda") for _ in range(2)]
        scales = [torch.zeros(1, rows, hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k, v, *pools, *scales)
        k, v = kv8_read(*pools, *scales, torch.zeros(1, **INT), rows, dtype=FP32)
    else:
        pools = [k.to(store), v.to(store)]
        k, v = (p.float() for p in pools)
    got, lse = gqa_tree_decode(q, *pools, torch.tensor([prefix], **INT), prefix, k_scales=scales[0], v_scales=scales[1],
                               round_to_bfloat16=False, want_lse=True)
    score = torch.einsum("nhd,hd->nh", q[0].double(), k[0, token].double().repeat_interleave(hq // hkv, 0)) / math.sqrt(dim)
    far = score.abs() > 2.0 ** (power - 14)   # above or below all others by far, and not by the rounding of its sum
    assert far.double().mean() > 0.98
    want, mean, want_lse = tree_attention(q[0].double(), k[0].double(), v[0].double(), prefix, list(range(-1, nodes - 1)))
    # weights rounded to bf16 or better (2^-8 of a mean of |v|), the result rounded once
    off, bound = (got[0].double() - want).abs(), mean * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -8 * 1.01 * want.abs() + 1e-30
    assert (off <= bound)[far].all(), (off / bound)[far].max().item()
    assert ((lse[0].double() - want_lse).abs() <= 2e-5 * want_lse.abs().clamp(min=1))[far].all()
    assert _capi.kernel_status() == 0
