"""Packed attention's kernel of two tiles that share their keys, over prompts of thousands of rows, against the definition in f64; each
case is first captured, to see that it is that kernel which it reaches."""
import pytest
import torch

from captured import kernels_of
from test_packed_attend_gpu import agree, attend_of, case, i32, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    o.stream(0)  # tensors of these tests live on the default stream
    yield o
    o.close()


def kernel_of(ops, path, q, k, v, ptr, hq, hk, d):
    at, out = i32(ptr), torch.empty(q.shape[0], hq * d, dtype=torch.bfloat16, device="cuda")
    names = kernels_of(ops, path, lambda: ops.packed_attend(q, k, v, at, hq, hk, d, 0.1, out))
    ops.stream(0)
    assert len(names) == 1
    return "pairs" if "paired_kernel" in names[0] else "single" if "single_kernel" in names[0] else names[0]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(32, 16), (64, 16), (48, 8), (64, 2)])
@pytest.mark.parametrize("lens,before,behind", [([2048], 0, 0), ([2049], 0, 3), ([2175], 1, 0), ([2304], 0, 100), ([2431, 0, 4096], 7, 0), ([4099, 1, 2560], 0, 9)])
def test_prompts_of_thousands_in_pairs(ops, tmp_path, lens, before, behind, hq, hk, d):
    q, k, v, ptr = case(hq, hk, d, lens, seed=len(lens) + hq, before=before, behind=behind)
    assert kernel_of(ops, tmp_path / "graph", q, k, v, ptr, hq, hk, d) == "pairs"
    agree(run(ops, q, k, v, ptr, hq, hk, d, d ** -0.5), *attend_of(q, k, v, ptr, hq, hk, d, d ** -0.5), ptr)


@pytest.mark.parametrize("hq,hk,d,lens", [(16, 8, 128, [5000]), (16, 8, 128, [5003, 17, 3000]), (32, 8, 128, [8192]), (24, 4, 64, [7001])])
def test_long_prompts_in_pairs(ops, tmp_path, hq, hk, d, lens):
    q, k, v, ptr = case(hq, hk, d, lens, seed=hq)
    assert kernel_of(ops, tmp_path / "graph", q, k, v, ptr, hq, hk, d) == "pairs"
    agree(run(ops, q, k, v, ptr, hq, hk, d, d ** -0.5), *attend_of(q, k, v, ptr, hq, hk, d, d ** -0.5), ptr)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(32, 16), (64, 16)])
def test_other_rows_do_not_reach_a_row_in_pairs(ops, tmp_path, hq, hk, d):
    """NaN and infinities in rows of no sequence, in the sequence behind and in later rows of the same sequence."""
    nan, inf, lens, before = float("nan"), float("inf"), [2300, 2090, 2200], 5
    q, k, v, ptr = case(hq, hk, d, lens, seed=3, before=before, behind=60)
    assert kernel_of(ops, tmp_path / "graph", q, k, v, ptr, hq, hk, d) == "pairs"
    for x in (q, k, v):
        x[:before], x[int(ptr[-1]):] = nan, inf
    k[int(ptr[1]):int(ptr[2])] = nan          # the whole second sequence
    v[int(ptr[1]):int(ptr[2])] = -inf
    late = lens[0] // 128 * 128               # rows of the first: in its last block,
    v[int(ptr[0]) + late + 34, 7] = nan
    v[int(ptr[0]) + late + 14, 9] = inf
    v[int(ptr[0]) + late + 15, 9] = -inf
    v[int(ptr[1]) - 1, d * (hk - 1) + 11] = -inf
    v[int(ptr[2]) + 100, 13] = inf            # and in one that later rows see as a whole
    v[int(ptr[3]) - 1, 3] = nan
    want, tol = attend_of(q, k, v, ptr, hq, hk, d, 0.1)
    want[int(ptr[1]):int(ptr[2])] = nan
    agree(run(ops, q, k, v, ptr, hq, hk, d, 0.1), want, tol, ptr)


@pytest.mark.parametrize("hq,hk,lens", [(16, 8, [77]), (4, 2, [4096]), (5, 1, [8192]), (32, 8, [100] * 60)])
def test_what_is_not_for_pairs(ops, tmp_path, hq, hk, lens):
    """Too little work for every SM, groups of an odd number, sequences shorter than two items."""
    q, k, v, ptr = case(hq, hk, 128, lens)
    assert kernel_of(ops, tmp_path / "graph", q, k, v, ptr, hq, hk, 128) == "single"
