"""The prepare step of drafted tokens: parents out of range, and nodes that a sequence does not have."""
import pytest
import torch

from pluto_b200 import _capi
from pluto_b200.layers import draft_prepare

pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


def prepare(parents, counts=None, store=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q, k, v = rnd(2, 4, 4, 64).bfloat16(), rnd(2, 4, 2, 64).bfloat16(), rnd(2, 4, 2, 64).bfloat16()
    pools = [torch.zeros(2, 16, 2, 64, dtype=store, device="cuda") for _ in range(2)]
    out = draft_prepare(q, k, v, rnd(64) * 0.1, rnd(64) * 0.1, torch.tensor([5, 3], **INT), *pools, rotary_dim=32,
                        parents=None if parents is None else torch.tensor(parents, **INT),
                        counts=None if counts is None else torch.tensor(counts, **INT))
    return [out] + pools


@pytest.mark.parametrize("bad", [-2, -9, -2 ** 31, 2, 3, 7, 2 ** 31 - 1])
def test_parents_out_of_range_are_reported_and_taken_as_first_tokens(bad):
    got = prepare([[-1, 0, 1, 2], [-1, 0, bad, 2]])
    assert _capi.kernel_status() & 0xff == 5
    want = prepare([[-1, 0, 1, 2], [-1, 0, -1, 2]])
    assert _capi.kernel_status() == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_queries_of_nodes_that_a_sequence_does_not_have_are_zeros():
    want = prepare(None)[0]
    torch.use_deterministic_algorithms(True)   # (new memory then holds NaN)
    try:
        got = prepare(None, counts=[4, 1])[0]
    finally:
        torch.use_deterministic_algorithms(False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :1], want[1, :1]) and not got[1, 1:].any()
    assert _capi.kernel_status() == 0
