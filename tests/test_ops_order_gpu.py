"""Calls made one behind the other on one stream, without waits: what one writes, the next reads."""
import numpy as np
import pytest
import torch

from captured import kernels_of

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def ops(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    o.stream(0)  # tensors of these tests live on the default stream
    yield o
    o.close()


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


def empty(*shape):
    return torch.full(shape, -1, dtype=torch.int32, device="cuda")


class Server:
    """Sequences that grow by `add` tokens a call, whose tables the device makes in place, over a bf16 cache."""
    HQ, HK, D = 4, 2, 128

    def __init__(self, n, add, steps):
        rng = np.random.default_rng(n)
        self.rows, width = sum(add), max(add) * steps // PAGE + 2
        total = n * width
        self.lens, self.add, self.table = i32(np.zeros(n)), i32(add), empty(n, width)
        self.free, self.count = i32(rng.permutation(total)), i32([total])
        self.indptr, self.pages, self.row_ptr, self.status = empty(n + 1), empty(total), empty(n + 1), empty(1)
        self.pos, self.slot, self.seq = empty(self.rows), empty(self.rows), empty(self.rows)
        self.kv = torch.zeros((total, self.HK, 2, PAGE, self.D), dtype=torch.bfloat16, device="cuda")
        g = torch.Generator(device="cuda")
        g.manual_seed(n)
        self.qkv = torch.randn(steps, self.rows, (self.HQ + 2 * self.HK) * self.D, generator=g, device="cuda").to(torch.bfloat16)
        self.gain = torch.ones(self.D, dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros(steps, self.rows, self.HQ * self.D, dtype=torch.bfloat16, device="cuda")

    def tables(self, ops):
        ops.kv_tables(self.lens, self.add, self.table, self.free, self.count, self.lens, self.count, self.indptr, self.pages, self.row_ptr,
                      self.pos, self.slot, self.seq, self.status)

    def attend(self, ops, t, prompt):
        ops.rope_attend(self.qkv[t], self.gain, self.gain, self.kv, self.kv.shape[0], self.pos, self.slot, self.seq if prompt else None,
                        self.indptr, self.pages, self.HQ, self.HK, self.D, 1e-6, 1e6, self.out[t])


def test_calls_that_read_ahead_stand_behind_all(ops, tmp_path):
    """Kernels that read positions, slots, counts or draws before they wait for the kernel in front have one in front that everything
    before it has to end for, whatever wrote them."""
    s = Server(3, [1, 1, 1], 2)
    logits = torch.zeros(3, 64, dtype=torch.bfloat16, device="cuda")
    uniforms, words, codes = torch.zeros(3, 16, device="cuda"), empty(3, 17), empty(3, 16)
    state, drawn = torch.zeros(3, 4096, dtype=torch.uint8, device="cuda"), empty(3, 17)
    reads_early = [
        ("rope_kv_kernel", lambda: s.attend(ops, 0, False)),
        ("rope_kv_kernel", lambda: s.attend(ops, 0, True)),
        ("sample_kernel", lambda: ops.sample(logits, 0.9, 0, 1.0, 1.0, 0, 0, -1, 0, s.lens, uniforms, words, state, s.seq, 4096, 0, 0, codes, 0)),
        ("lm_sample_kernel", lambda: ops.lm_sample(logits, 0.8, 1, words, s.table, 0, drawn)),
    ]
    for name, call in reads_early:
        def calls(call=call):
            s.tables(ops)
            call()
        names = kernels_of(ops, tmp_path / "graph", calls)
        at = next(i for i, k in enumerate(names) if name in k)
        assert "kv_tables_kernel" in names[0] and any("order_kernel" in k for k in names[1:at]), names


@pytest.mark.parametrize("n,add,prompt", [(5, 1, False), (64, 1, False), (700, 1, False), (64, 1, True), (40, 23, True)])
def test_tables_then_attention_over_bf16_pages(ops, n, add, prompt):
    """Tables made on the device and the bf16 attention that reads them, call after call: as if every call were waited for."""
    steps, got = 20, []
    for wait in (True, False):
        s = Server(n, [add] * n, steps)
        torch.cuda.synchronize()
        for t in range(steps):
            s.tables(ops)
            if wait:
                ops.sync()
            s.attend(ops, t, prompt)
            if wait:
                ops.sync()
        ops.sync()
        assert s.status.item() == 0 and s.lens.tolist() == [add * steps] * n
        got.append((s.kv, s.out, s.qkv))
    for waited, chained in zip(*got):
        assert torch.equal(waited, chained)
