"""Arguments that the operators' documentation allows."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    o.stream(0)  # tensors of these tests live on the default stream
    yield o
    o.close()


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("wider", [0, 8, 512])
def test_norm_and_rope_in_place_on_parts_of_wider_rows(ops, rows, wider):
    """q and k rotated where they lie, given as all of a projection's row and as its first part."""
    hq, hk, d = 4, 2, 64
    width = (hq + hk) * d
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    x = torch.randn(rows, width + wider, generator=g, device="cuda").to(torch.bfloat16)
    gain = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    pos = torch.tensor(np.arange(rows) * 7, dtype=torch.int32, device="cuda")
    want = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope(x, gain, gain, pos, hq, hk, d, 1e-6, 1e4, want)
    rest = x[:, width:].clone()
    ops.qk_norm_rope(x, gain, gain, pos, hq, hk, d, 1e-6, 1e4, x[:, :width])
    ops.sync()
    assert torch.equal(x[:, :width], want) and torch.equal(x[:, width:], rest)


def test_an_error_is_reported_once(ops):
    """A context for a device that is not there is refused; the calls behind it do not hear of it again."""
    from pega_omni_b200.ops import Ops, OpsError
    w, x = (torch.randn(*shape, device="cuda").to(torch.bfloat16) for shape in ((64, 128), (2, 128)))
    y = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    for again in range(2):
        with pytest.raises(OpsError, match="device"):
            Ops(99)
        ops.chain_gemm(w, x, y)
        ops.sync()
    assert y.abs().sum() > 0
