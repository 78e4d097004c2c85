"""Device lengths that run past the end of a sequence's only page, whose size no step or tile of the kernels divides."""
import pytest
import torch

from drafts_double import tree_attention
from pluto_b200 import _capi
from pluto_b200.layers import gqa_tree_decode, kv8_append, kv8_read

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")
EIGHT, BF16, FP32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


@pytest.mark.parametrize("store", [EIGHT, BF16, FP32])
@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("size,prefix", [(20, 18), (20, 17), (20, 27), (20, 40), (7, 5), (21, 18), (77, 75)])
@pytest.mark.parametrize("hq,hkv,dim", [(4, 2, 128), (4, 4, 64), (4, 4, 256), (8, 2, 64), (16, 2, 128), (12, 2, 256), (80, 2, 64)])
def test_slots_behind_the_page_read_as_zeros_and_are_reported(store, table, size, prefix, hq, hkv, dim):
    """The rows of the sequence behind it, and the bytes behind the pool, hold NaN and scale bytes of 255."""
    nodes, pages = 4, 4   # sequences 0 and 2 take part, 1 does not, page 3 is nobody's
    gen = torch.Generator(device="cuda").manual_seed(size + dim)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    k, v, q = rnd(pages, size, hkv, dim), rnd(pages, size, hkv, dim), rnd(3, nodes, hq, dim).bfloat16()
    scales = []
    if store == EIGHT:
        rows = [torch.zeros(pages, size, hkv, dim, dtype=store, device="cuda") for _ in range(2)]
        scales = [torch.zeros(pages, size, hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
        kv8_append(k, v, *rows, *scales)
        k, v = kv8_read(*rows, *scales, torch.zeros(pages, **INT), size, dtype=FP32)
    else:
        rows = [k.to(store), v.to(store)]
        k, v = (r.float() for r in rows)
    for r in rows:
        bad = r.view(torch.uint8) if store == EIGHT else r
        bad[1], bad[3] = (0x7f, 0x7f) if store == EIGHT else (float("nan"), float("nan"))
    for s in scales:
        s[1] = s[3] = 255
    blocks = torch.tensor([[0], [1], [2]], **INT) if table else None
    if not table:   # the pool ends where the guard begins
        rows, scales = [r[:3] for r in rows], [s[:3] for s in scales]
    got = gqa_tree_decode(q, *rows, torch.tensor([prefix, 0, prefix], **INT), prefix, counts=torch.tensor([nodes, 0, nodes], **INT),
                          block_table=blocks, k_scales=scales[0] if scales else None, v_scales=scales[1] if scales else None,
                          round_to_bfloat16=False)
    assert _capi.kernel_status() & 0xff == 2
    none = torch.zeros(max(0, prefix + nodes - size), hkv, dim, device="cuda")
    for b in (0, 2):
        kk, vv = (torch.cat([x[b], none])[:prefix + nodes].double() for x in (k, v))
        want, mean, _ = tree_attention(q[b].double(), kk, vv, prefix, list(range(-1, nodes - 1)))
        # weights rounded to bf16 or better (2^-8 of a mean of |v|), the result rounded once
        off, bound = (got[b].double() - want).abs(), mean * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -8 * 1.01 * want.abs() + 1e-30
        assert (off <= bound).all(), (b, (off / bound).max().item())
    assert not got[1].any()
