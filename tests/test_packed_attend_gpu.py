"""Causal attention over packed prompts on the GPU against its definition in f64, and the operators of the 8-bit cache together as a
server runs them."""
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


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


def bf16(x):
    return torch.as_tensor(np.asarray(x, dtype=np.float32)).to(torch.bfloat16).cuda()


def packed(lens, before=0, behind=0):
    return np.concatenate([[before], before + np.cumsum(lens)]).astype(np.int32), before + int(np.sum(lens)) + behind


def attend_of(q, k, v, ptr, hq, hk, d, scale):
    """(result, tolerance) in f64 on the GPU; rows of no sequence: NaN. Values that are not finite count for the rows that see them."""
    q, k, v = q.double(), k.double(), v.double()
    rows = q.shape[0]
    out, tol = (torch.full((rows, hq * d), float("nan"), dtype=torch.float64, device="cuda") for _ in range(2))
    for a, b in zip(ptr, ptr[1:]):
        n = int(b - a)
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(hq):
            g = h // (hq // hk)
            qh, kh, vh = q[a:b, h * d:(h + 1) * d], k[a:b, g * d:(g + 1) * d], v[a:b, g * d:(g + 1) * d]
            s = (qh @ kh.T) * scale
            w = torch.softmax(s.masked_fill(hidden, -float("inf")), -1)
            fine = vh.isfinite()
            o = w @ torch.where(fine, vh, 0)
            # what is not finite: reaches rows from its own on
            seen = lambda m: m.to(torch.int64).cumsum(0) > 0  # noqa: E731
            up, down, nan = seen(vh == float("inf")), seen(vh == -float("inf")), seen(vh.isnan())
            o = torch.where(nan | (up & down), float("nan"), torch.where(up, float("inf"), torch.where(down, -float("inf"), o)))
            # the result's rounding and the weights' (2^-8 each); their exponents: a score is a sum of d products, every addition off by 2^-23 of
            # the magnitudes at most, times a product of f32; ex2 and f32 sums over n keys
            mag = (qh.abs() @ torch.where(kh.isfinite(), kh, 0).abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True) * scale
            r = 2.0 ** -8 + 2 * (d + 4) * 2.0 ** -23 * mag + (n / 2 + 8) * 2.0 ** -23
            out[a:b, h * d:(h + 1) * d] = o
            tol[a:b, h * d:(h + 1) * d] = o.abs() * 2.0 ** -8 + (w @ torch.where(fine, vh, 0).abs()) * r * (1 + 2.0 ** -7) + 1e-38
    return out, tol


def run(ops, q, k, v, ptr, hq, hk, d, scale):
    out = torch.full((q.shape[0], hq * d + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.packed_attend(q, k, v, i32(ptr), hq, hk, d, scale, out[:, :hq * d])
    ops.sync()
    assert (out[:, hq * d:] == 3).all()
    return out[:, :hq * d]


def agree(got, want, tol, ptr):
    inside = torch.zeros(got.shape[0], dtype=torch.bool, device="cuda")
    inside[int(ptr[0]):int(ptr[-1])] = True
    assert (got[~inside] == 3).all(), "a row of no sequence was written"
    got, want, tol = got[inside].double(), want[inside], tol[inside]
    fine = want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(7, 8, 9), want[~fine].nan_to_num(7, 8, 9))
    off = ((got - want).abs() / tol)[fine]
    assert off.numel() == 0 or off.max() <= 1, (off.max().item(), torch.argwhere(((got - want).abs() > tol) & fine)[:4].tolist())


def case(hq, hk, d, lens, seed=0, before=0, behind=0, loud=1.0):
    ptr, rows = packed(lens, before, behind)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    qkv = (torch.randn(rows, (hq + 2 * hk) * d, generator=g, device="cuda") * loud).to(torch.bfloat16)
    return qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:], ptr


def check(ops, hq, hk, d, lens, scale=None, **kw):
    q, k, v, ptr = case(hq, hk, d, lens, **kw)
    scale = d ** -0.5 if scale is None else scale
    agree(run(ops, q, k, v, ptr, hq, hk, d, scale), *attend_of(q, k, v, ptr, hq, hk, d, scale), ptr)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (5, 1)])
@pytest.mark.parametrize("n", [1, 2, 31, 64, 127, 128, 129, 255, 256, 257, 384, 385, 700])
def test_one_prompt(ops, n, hq, hk, d):
    check(ops, hq, hk, d, [n], seed=n)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(3, 3), (4, 2), (6, 2), (16, 8), (16, 1)])
@pytest.mark.parametrize("lens,before,behind", [
    ([1, 1, 1], 0, 0), ([0, 5, 0, 0, 130, 0], 0, 0), ([77, 128, 129, 3], 0, 19), ([200, 300], 41, 0), ([0], 0, 6), ([0, 0], 7, 7), ([257, 1, 256, 255], 1, 128),
])
def test_packed_prompts(ops, lens, before, behind, hq, hk, d):
    check(ops, hq, hk, d, lens, seed=len(lens), before=before, behind=behind)


def test_many_prompts(ops):
    """More sequences than a block has threads."""
    lens = np.random.default_rng(0).integers(0, 40, 1000).tolist()
    check(ops, 2, 1, 64, lens, behind=3)
    check(ops, 3, 1, 64, lens)


@pytest.mark.parametrize("d,n", [(128, 2500), (64, 5000)])
def test_long_prompts(ops, d, n):
    check(ops, 2, 1, d, [n])
    check(ops, 1, 1, d, [n, 3])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (3, 1), (4, 2)])
@pytest.mark.parametrize("lens,before,behind", [([2048], 0, 0), ([2049], 0, 3), ([2175], 1, 0), ([2177], 0, 0), ([2304], 0, 100), ([2431, 0, 4096], 7, 0), ([4099, 1, 2560], 0, 9)])
def test_prompts_of_thousands(ops, lens, before, behind, hq, hk, d):
    """Sequences long enough in the mean for the kernel that shares keys between two tiles of queries."""
    check(ops, hq, hk, d, lens, seed=len(lens), before=before, behind=behind)


@pytest.mark.parametrize("scale", [1e-38, 1e-3, 2.0])  # 0 is refused: a hidden score is -infinity before it is scaled
@pytest.mark.parametrize("loud", [0.05, 3.0])
def test_flat_and_peaked(ops, scale, loud):
    """Equal weights; rows that one key has to itself; references that rise from block to block."""
    check(ops, 2, 1, 128, [520], scale=scale, loud=loud)
    q, k, v, ptr = case(2, 2, 64, [900], seed=9)
    k = (k.float() * torch.linspace(0.01, 4, 900, device="cuda")[:, None]).to(torch.bfloat16)
    agree(run(ops, q, k, v, ptr, 2, 2, 64, scale), *attend_of(q, k, v, ptr, 2, 2, 64, scale), ptr)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(2, 1), (1, 1)])
@pytest.mark.parametrize("lens", [[300, 90, 200], [2300, 2090, 2200]])
def test_other_rows_do_not_reach_a_row(ops, lens, hq, hk, d):
    """NaN and infinities in rows of no sequence, in the sequence behind and in later rows of the same sequence."""
    before, behind = 5, 60
    nan, inf = float("nan"), float("inf")
    q, k, v, ptr = case(hq, hk, d, lens, seed=3, before=before, behind=behind)
    for x in (q, k, v):
        x[:before], x[int(ptr[-1]):] = nan, inf
    k[int(ptr[1]):int(ptr[2])] = nan          # the whole second sequence
    v[int(ptr[1]):int(ptr[2])] = -inf
    late = lens[0] // 128 * 128               # rows of the first: in its last block,
    v[int(ptr[0]) + late + 34, 7] = nan
    v[int(ptr[0]) + late + 14, 9] = inf
    v[int(ptr[0]) + late + 15, 9] = -inf
    v[int(ptr[1]) - 1, 11] = -inf
    v[int(ptr[2]) + 100, 13] = inf            # and in one that later rows see as a whole
    v[int(ptr[3]) - 1, 3] = nan
    want, tol = attend_of(q, k, v, ptr, hq, hk, d, 0.1)
    want[int(ptr[1]):int(ptr[2])] = nan
    got = run(ops, q, k, v, ptr, hq, hk, d, 0.1)
    assert (got[:before] == 3).all() and (got[int(ptr[-1]):] == 3).all()
    agree(got, want, tol, ptr)
    # a key that is no number takes the rows from its own on
    q, k, v, ptr = case(hq, hk, d, [400], seed=4)
    k[350, 1] = nan
    want, tol = attend_of(q, k, v, ptr, hq, hk, d, 0.1)
    got = run(ops, q, k, v, ptr, hq, hk, d, 0.1)
    assert got[350:].isnan().all()
    agree(got[:350], want[:350], tol[:350], [0, 350])


def test_rows_of_their_own_stride(ops):
    """q, k, v and out in buffers of their own, rows wider than the heads."""
    hq, hk, d, n = 4, 2, 128, 333
    q, k, v, ptr = case(hq, hk, d, [n], seed=6)
    wide = [torch.cat([x, torch.full((n, 8 * (i + 1)), float("nan"), dtype=torch.bfloat16, device="cuda")], 1) for i, x in enumerate((q, k, v))]
    parts = [w[:, :x.shape[1]] for w, x in zip(wide, (q, k, v))]
    agree(run(ops, *parts, ptr, hq, hk, d, 0.09), *attend_of(q, k, v, ptr, hq, hk, d, 0.09), ptr)


@pytest.mark.parametrize("ptr", [[0, 41], [-1, 20], [30, 10, 20], [0, 10, 2**31 - 1]])
def test_sequences_outside_the_rows_are_reported(ops, ptr):
    from pega_omni_b200.ops import OpsError
    q, k, v, _ = case(2, 1, 64, [40])
    out = torch.zeros((40, 128), dtype=torch.bfloat16, device="cuda")
    ops.packed_attend(q, k, v, i32(ptr), 2, 1, 64, 0.1, out)
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()


@pytest.mark.parametrize("hq,hk,d", [(4, 1, 64), (8, 1, 128), (16, 1, 64), (32, 1, 128), (48, 2, 64), (12, 1, 128), (20, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("lens", [[9, 1, 0, 70, 8, 17], [300, 129, 64, 65, 5], [1] * 40, [700, 33]])
def test_heads_that_share_a_tile(ops, hq, hk, d, lens):
    """Groups of all sizes, whose heads share tiles: what is not finite reaches the rows behind it in each head alike."""
    check(ops, hq, hk, d, lens, seed=hq, before=3, behind=5)
    q, k, v, ptr = case(hq, hk, d, lens, seed=hq + 1)
    at = int(ptr[1]) - 1 - (15 if lens[0] > 20 else 0)  # of the first sequence
    v[at, 3], v[at, 5], v[int(ptr[0]), 7] = float("nan"), -float("inf"), float("inf")
    agree(run(ops, q, k, v, ptr, hq, hk, d, 0.1), *attend_of(q, k, v, ptr, hq, hk, d, 0.1), ptr)


@pytest.mark.parametrize("hq,hk,d", [(64, 32, 128), (64, 16, 64), (96, 16, 64), (48, 2, 128), (64, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("lens", [[300, 257, 513, 260], [700, 1000, 0, 333], [1, 2050, 3], [384] * 5])
@pytest.mark.parametrize("odd", [False, True])
def test_tiles_in_pairs(ops, hq, hk, d, lens, odd):
    """As many heads as it takes for two tiles a block: sizes around its tiles, what is not finite, rows of nobody."""
    q, k, v, ptr = case(hq, hk, d, lens, seed=hq + d, before=2, behind=9)
    if odd:
        for x in (q, k, v):
            x[:2], x[int(ptr[-1]):] = float("nan"), float("inf")
        last = int(ptr[2]) - 1  # of the second sequence
        v[last, 3], v[last - 9, 5], v[last - 200 if lens[1] > 200 else last, 7], v[last - 1, 5] = float("nan"), -float("inf"), float("inf"), float("inf")
        v[int(ptr[0]), d - 1] = float("nan")
    agree(run(ops, q, k, v, ptr, hq, hk, d, 0.1), *attend_of(q, k, v, ptr, hq, hk, d, 0.1), ptr)


def test_sequences_over_one_another_end(ops):
    """Many sequences of all the rows: more work than rows and sequences can make is not begun."""
    from pega_omni_b200.ops import OpsError
    q, k, v, _ = case(2, 1, 64, [1000])
    out = torch.full((1000, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.packed_attend(q, k, v, i32([0, 1000] * 20), 2, 1, 64, 0.1, out)
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()
    assert (out == 3).all()


@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 2)])
@pytest.mark.parametrize("lens", [[1900, 3, 700, 3, 130, 0, 1400], [3] * 70 + [4000] + [129] * 3, [128] * 300, [4000] + [0] * 40 + [2600]])
def test_prompts_of_all_lengths(ops, hq, hk, lens):
    """One long sequence among many short ones, lengths that many have, empty ones between."""
    check(ops, hq, hk, 64, lens, seed=len(lens))


@pytest.mark.parametrize("lens", [[300, 77, 512], [5000]])
def test_the_same_every_time_and_from_a_graph(ops, lens):
    q, k, v, ptr = case(16, 8, 128, lens, seed=8)
    want = run(ops, q, k, v, ptr, 16, 8, 128, 0.1).clone()
    stream, graph, at = torch.cuda.Stream(), torch.cuda.CUDAGraph(), i32(ptr)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.stream(stream.cuda_stream)
        ops.packed_attend(q, k, v, at, 16, 8, 128, 0.1, out)
    ops.stream(0)
    for _ in range(10):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_side_by_side(ops):
    """Calls of both kernels and both head sizes on streams of their own, all under way at once."""
    cases = [(16, 8, 128, [5000]), (16, 8, 128, [300, 77, 512]), (64, 32, 64, [700, 300]), (4, 4, 64, [64] * 50), (5, 1, 128, [2000, 9])]
    graphs, streams, outs, want, held = [], [], [], [], []
    for n, (hq, hk, d, lens) in enumerate(cases):
        q, k, v, ptr = case(hq, hk, d, lens, seed=n)
        want.append(run(ops, q, k, v, ptr, hq, hk, d, 0.1).clone())
        held.append((q, k, v, i32(ptr)))
        outs.append(torch.zeros_like(want[-1], memory_format=torch.contiguous_format))
        streams.append(torch.cuda.Stream())
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1], stream=streams[-1]):
            ops.stream(streams[-1].cuda_stream)
            for _ in range(3):
                ops.packed_attend(*held[-1], hq, hk, d, 0.1, outs[-1])
        ops.stream(0)
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    ops.sync()


# ---- together ---------------------------------------------------------------------------------------------------------------

def plain_rope(x, gain, pos, d, theta):
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain.double()
    a = pos.double()[:, None, None] * theta ** (-2 * torch.arange(d // 2, dtype=torch.float64, device="cuda") / d)
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)


@pytest.mark.parametrize("hq,hk,d,n", [(16, 8, 128, 24), (10, 2, 64, 3), (16, 1, 128, 70)])
def test_calls_behind_one_another(ops, hq, hk, d, n):
    """Steps in which every call takes what the one in front has written give the same with and without a wait between the calls."""
    rng = np.random.default_rng(n)
    steps, width, prompt = 12, 40, 60
    adds = [i32(rng.integers(1, prompt, n))] + [i32(rng.choice([-1, 0, 1, 1, 1], n) if k % 4 == 3 else np.ones(n)) for k in range(1, steps)]
    rows = [prompt * n] + [n] * (steps - 1)
    xs = [bf16(rng.standard_normal((r, (hq + 2 * hk) * d))) for r in rows]
    gain = bf16(1 + 0.1 * rng.standard_normal(d))

    def go(wait):
        outs = []
        done = torch.cuda.synchronize if wait else lambda: None
        lens, count, free, table = i32([0] * n), i32([n * width]), i32(np.arange(n * width)), i32(np.zeros((n, width)))
        kv, scales = torch.zeros((n * width, hk, 2, 16, d), dtype=torch.uint8, device="cuda"), torch.ones((n * width, hk, 2), device="cuda")
        indptr, row_ptr, pages, status = i32([0] * (n + 1)), i32([0] * (n + 1)), i32([0] * (n * width)), i32([0])
        pos, slot, seq = (i32([0] * max(rows)) for _ in range(3))
        states = [x.clone() for x in xs]
        torch.cuda.synchronize()
        for k, r in enumerate(rows):
            x, out = states[k], torch.full((r, hq * d), 2.0, dtype=torch.bfloat16, device="cuda")
            at = pos[:r], slot[:r], seq[:r]
            ops.kv_tables(lens, adds[k], table, free, count, lens, count, indptr, pages, row_ptr, *at, status), done()
            ops.qk_norm_rope(x, gain, gain, at[0], hq, hk, d, 1e-6, 1e6, x), done()
            q, key, v = x[:, :hq * d], x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:]
            ops.kv8_append(key, v, at[1], kv, scales), done()
            if k == 0:
                ops.packed_attend(q, key, v, row_ptr, hq, hk, d, 0.1, out), done()
            else:
                ops.kv8_attend(q, kv, scales, at[0], indptr, pages, hq, 0.1, out, at[2]), done()
            outs += [x, out]
        ops.sync()
        return outs + [lens, count, table, kv, scales, status]

    want = go(True)
    for _ in range(6):
        for a, b in zip(go(False), want):
            assert torch.equal(a.view(torch.int16) if a.dtype is torch.bfloat16 else a, b.view(torch.int16) if b.dtype is torch.bfloat16 else b)


@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (10, 2, 64)])
def test_a_server_runs_them_together(ops, hq, hk, d):
    """Prompts come, sequences step and end, others take their pages; the steps are one captured graph. Every row's attention is that
    of its sequence's whole history, to what 8 bits keep of it."""
    rng = np.random.default_rng(1)
    n, width, total, rows_max, theta = 6, 12, 40, 400, 1e6
    kv = torch.full((total, hk, 2, 16, d), 0x7f, dtype=torch.uint8, device="cuda")  # NaN until written
    scales = torch.full((total, hk, 2), float("nan"), device="cuda")
    q_norm, k_norm = bf16(1 + 0.2 * rng.standard_normal(d)), bf16(1 + 0.2 * rng.standard_normal(d))
    lens, add, count = i32([0] * n), i32([0] * n), i32([total])
    free, table = i32(rng.permutation(total)), i32(np.full((n, width), -1))
    st = {k: i32(np.zeros(m)) for k, m in dict(indptr=n + 1, pages=total, row_ptr=n + 1, pos=rows_max, slot=rows_max, seq=rows_max, status=1).items()}
    qkv = torch.zeros((rows_max, (hq + 2 * hk) * d), dtype=torch.bfloat16, device="cuda")
    qk = torch.zeros((rows_max, (hq + hk) * d), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((rows_max, hq * d), dtype=torch.bfloat16, device="cuda")
    history = [[] for _ in range(n)]

    def call(prompts, rows):
        ops.kv_tables(lens, add, table, free, count, lens, count, st["indptr"], st["pages"], st["row_ptr"], st["pos"][:rows], st["slot"][:rows], st["seq"][:rows], st["status"])
        ops.qk_norm_rope(qkv[:rows], q_norm, k_norm, st["pos"][:rows], hq, hk, d, 1e-6, theta, qk[:rows])
        k, v = qk[:rows, hq * d:], qkv[:rows, (hq + hk) * d:]
        ops.kv8_append(k, v, st["slot"][:rows], kv, scales)
        if prompts:
            ops.packed_attend(qk[:rows, :hq * d], k, v, st["row_ptr"], hq, hk, d, d ** -0.5, out[:rows])
        else:
            ops.kv8_attend(qk[:rows, :hq * d], kv, scales, st["pos"][:rows], st["indptr"], st["pages"], hq, d ** -0.5, out[:rows], st["seq"][:rows])

    def rows_of(adds):
        qkv.copy_(torch.from_numpy(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)))
        add.copy_(i32(adds))
        out.fill_(5)
        torch.cuda.synchronize()

    def check_call(adds, prompts, rows):
        torch.cuda.synchronize()
        ops.sync()
        assert st["status"].item() == 0
        r = 0
        for s, a in enumerate(adds):
            if a == -1:
                history[s] = []
            for _ in range(max(a, 0)):
                history[s].append(qkv[r].clone())
                x = torch.stack(history[s]).reshape(-1, hq + 2 * hk, d)
                pos = torch.arange(len(x), device="cuda")
                k, v = plain_rope(x[:, hq:hq + hk], k_norm, pos, d, theta), x[:, hq + hk:].double()
                q = plain_rope(x[-1:, :hq], q_norm, pos[-1:], d, theta)[0]
                w = torch.softmax(torch.einsum("hd,thd->ht", q, k.repeat_interleave(hq // hk, 1)) * d ** -0.5, -1)
                v = v.repeat_interleave(hq // hk, 1)
                want = torch.einsum("ht,thd->hd", w, v)
                size = torch.einsum("ht,thd->hd", w, v.abs())
                # K in 8 bits (2^-4 of each value) moves a score by at most 2^-4 sum |q||k| scale, in fact by about a 1 / sqrt(d) of it, of
                # which six are taken; V by 2^-4; bf16 q, k, weights and results by 2^-7 together
                ds = torch.einsum("hd,thd->ht", q.square(), k.repeat_interleave(hq // hk, 1).square()).sqrt().amax(-1, keepdim=True) * d ** -0.5
                lossy = 0 if prompts else 2.0 ** -4
                tol = size * (lossy * (1 + 6 * ds) + 2.0 ** -7 * (1 + 6 * ds) + 2.0 ** -6)
                assert ((out[r].double().reshape(hq, d) - want).abs() <= tol).all(), (s, len(x), ((out[r].double().reshape(hq, d) - want).abs() / tol).max())
                r += 1
        if not prompts:
            assert (out[r:rows] == 0).all()
        assert (out[rows:] == 5).all()

    adds = [40, 0, 1, 130, 16, 0]
    rows_of(adds)
    call(True, 200)  # rows behind the last belong to nobody
    check_call(adds, True, 200)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.stream(stream.cuda_stream)
        call(False, 8)
    ops.stream(0)
    for step in range(20):
        adds = [1, 0, 1, 1, 1, 0]
        if step == 9:
            adds = [-1, 0, 1, -1, 0, 0]
        elif step > 9:
            adds = [0, 0, 1, 0, 1, 0]
        rows_of(adds)
        graph.replay()
        check_call(adds, False, 8)
    adds = [0, 100, 0, 0, 0, 77]  # over pages that others held
    rows_of(adds)
    call(True, 177)
    check_call(adds, True, 177)
    for _ in range(3):
        adds = [0, 1, 1, 0, 1, 1]
        rows_of(adds)
        graph.replay()
        check_call(adds, False, 8)
