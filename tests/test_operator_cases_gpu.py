"""The measurable cases of the operators (perf/operators.py): a pass runs on the stream that is current when it is made."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [{"kind": "tables", "n": 9, "ctx_min": 5, "ctx_max": 300, "fresh": 1, "prompt_min": 40, "prompt_max": 40, "done": 1},
         {"kind": "rope", "rows": 33, "far": 500, "hq": 4, "hk": 2, "d": 64},
         {"kind": "append", "n": 5, "ctx_min": 0, "ctx_max": 40, "add_min": 1, "add_max": 20, "hq": 4, "hk": 2, "d": 64},
         {"kind": "prompt", "n": 3, "len_min": 5, "len_max": 150, "pad": 3, "hq": 4, "hk": 2, "d": 128},
         {"kind": "attend8", "n": 5, "ctx_min": 0, "ctx_max": 700, "hq": 4, "hk": 2, "d": 128}]


@pytest.fixture(scope="module")
def cases(built_lib):
    m = importlib.import_module("perf.operators")
    m.own = True
    yield m
    m.own = False


def outputs(got):
    return [t.view(torch.uint8) if t.element_size() == 1 else t for t in (got.values() if isinstance(got, dict) else [got])]


def state(cases, case):
    return cases.prepare(case, 3)


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(outputs(got), want, strict=True))


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["kind"])
def test_a_pass_runs_on_the_current_stream(cases, case):
    st = state(cases, case)
    want = [t.clone() for t in outputs(cases.run(st))]
    torch.cuda.synchronize()
    # under another stream, behind what that has still to do
    st, src = state(cases, case), state(cases, case)
    for k, t in st.items():
        if isinstance(t, torch.Tensor) and t.dtype != torch.int32:
            t.zero_()
    pos = "pos" if case["kind"] in ("rope", "attend8") else "add" if case["kind"] == "tables" else "slot" if case["kind"] == "append" else None
    if pos:
        st[pos].fill_(0 if case["kind"] == "tables" else -1)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)
        for k, t in st.items():
            if isinstance(t, torch.Tensor):
                t.copy_(src[k])
        got = cases.run(st)
        got = [t.clone() for t in outputs(got)]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    # in a capture under a stream of its own
    st = state(cases, case)
    saved = {k: t.clone() for k, t in st.items() if isinstance(t, torch.Tensor)}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cases.run(st)
    assert all(torch.equal(st[k], t) for k, t in saved.items()), "ran outside of the capture"
    graph.replay()
    torch.cuda.synchronize()
    assert same(got, want)
    # and on the first one again
    st = state(cases, case)
    assert same(cases.run(st), want)
    torch.cuda.synchronize()
