"""Packed attention with scores of any size: softmax looks at their differences alone."""
import pytest
import torch

from test_packed_attend_gpu import agree, packed, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    o.stream(0)  # tensors of these tests live on the default stream
    yield o
    o.close()


def check(ops, hq, hk, d, lens, key, query):
    """Queries and keys of one element each, so that a score is one exact product."""
    ptr, rows = packed(lens)
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    q, k = (torch.zeros(rows, h, d, device="cuda") for h in (hq, hk))
    q[:, :, 3], k[:, :, 3] = query.view(-1, 1), key.view(-1, 1)
    q, k = q.flatten(1).to(torch.bfloat16), k.flatten(1).to(torch.bfloat16)
    v = torch.randn(rows, hk * d, generator=g, device="cuda").to(torch.bfloat16)
    scale = d ** -0.5
    want, tol = (torch.zeros(rows, hq * d, dtype=torch.float64, device="cuda") for _ in range(2))
    for a, b in zip(ptr, ptr[1:]):
        n = int(b - a)
        # equal keys have equal scores, bit for bit; those of others differ by much, or are off by a rounding of a difference below 2^14
        s = q[a:b, 3].double()[:, None] * k[a:b, 3].double()[None] * scale
        w = torch.softmax(s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -float("inf")), -1)
        r = 2.0 ** -8 + 2 * 2.0 ** -23 * 2.0 ** 14 + (n / 2 + 8) * 2.0 ** -23
        for h in range(hq):
            at, vh = slice(h * d, (h + 1) * d), v[a:b, h // (hq // hk) * d:(h // (hq // hk) + 1) * d].double()
            want[a:b, at] = w @ vh
            tol[a:b, at] = want[a:b, at].abs() * 2.0 ** -8 + (w @ vh.abs()) * r * (1 + 2.0 ** -7) + 1e-38
    agree(run(ops, q, k, v, ptr, hq, hk, d, scale), want, tol, ptr)


SIZES = [1.0, 3e3, 1e7, 3e9, 1e12, 1e20, 1e30, 2e37]


@pytest.mark.parametrize("hq,hk,d,lens", [(2, 1, 128, [1, 700, 3]), (5, 1, 64, [300, 129]), (32, 16, 128, [2050, 9, 2048]), (16, 1, 64, [90] * 20)])
@pytest.mark.parametrize("size", SIZES + [-s for s in SIZES])
def test_scores_of_any_size(ops, size, hq, hk, d, lens):
    """Two kinds of keys, of one or two times a size."""
    rows = sum(lens)
    high = torch.rand(rows, generator=torch.Generator().manual_seed(rows)).cuda() < 0.1
    check(ops, hq, hk, d, lens, torch.where(high, 2.0, 1.0), torch.full((rows,), size, device="cuda"))


@pytest.mark.parametrize("hq,hk,d,lens", [(2, 1, 128, [1500]), (5, 1, 64, [600, 900]), (32, 16, 128, [2050, 2048]), (16, 1, 64, [400] * 9)])
def test_scores_that_change_their_size(ops, hq, hk, d, lens):
    """From block to block from small ones to large ones and back, up and down, of either sign."""
    rows = sum(lens)
    size = torch.tensor([1.0, -1e12, 3.0, 1e9, -1e20, 1e12, 0.0, -1e10, 1e20], device="cuda")
    key = size[torch.arange(rows, device="cuda") // 70 % 9] * torch.where(torch.arange(rows, device="cuda") % 3 == 0, 2.0, 1.0)
    check(ops, hq, hk, d, lens, key, torch.where(torch.arange(rows, device="cuda") % 2 == 0, 1.0, -1.0))
