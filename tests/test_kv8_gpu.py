"""The operators around the 8-bit paged cache on the GPU, each against its definition in numpy (64 bits), and a run of them
together as a server makes it."""
import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 16
MIN_SCALE = 2.0 ** -100


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


def f64(t):
    return t.detach().cpu().double().numpy()


# ---- page tables ---------------------------------------------------------------------------------------------------------

def tables_of(lens, add, table, free, count):
    """What the call leaves, request by request."""
    lens, table, stack = list(lens), table.copy(), list(free[:count])
    indptr, row_ptr, pages, rows = [0], [0], [], []
    for s, a in enumerate(add):
        if a == -1:
            stack += list(table[s, :-(-lens[s] // PAGE)])
    for s, a in enumerate(add):
        total = 0 if a == -1 else lens[s] + a
        if a != -1:
            for p in range(-(-lens[s] // PAGE), -(-total // PAGE)):
                table[s, p] = stack.pop()
        pages += list(table[s, :-(-total // PAGE)])
        rows += [(p, table[s, p // PAGE] * PAGE + p % PAGE, s) for p in range(lens[s], total)]
        indptr.append(len(pages)), row_ptr.append(len(rows))
        lens[s] = total
    return lens, stack, table, indptr, pages, row_ptr, rows


class Tables:
    """Device arrays of a call, with guards where nothing may be written."""

    def __init__(self, lens, add, width, spare, row_cap=None, page_cap=None, free_cap=None, seed=0):
        rng = np.random.default_rng(seed)
        n = len(lens)
        held = [-(-c // PAGE) for c in lens]
        ids = rng.permutation(sum(held) + spare).astype(np.int32)
        self.table0 = np.full((n, width), -7, dtype=np.int32)
        at = 0
        for s, h in enumerate(held):
            self.table0[s, :h] = ids[at:at + h]
            at += h
        self.free0 = np.full(sum(held) + spare if free_cap is None else free_cap, -9, dtype=np.int32)
        self.free0[:spare] = ids[at:]
        self.lens0, self.add0, self.spare = list(lens), list(add), spare
        rows = sum(max(a, 0) for a in add)
        pages = sum(0 if a == -1 else -(-(c + a) // PAGE) for c, a in zip(lens, add))
        self.rows, self.pages_n = rows, pages
        self.lens, self.add, self.table, self.free, self.count = i32(lens), i32(add), i32(self.table0), i32(self.free0), i32([spare])
        full = lambda k: i32(np.full(k, -5))  # noqa: E731
        self.indptr, self.row_ptr, self.status = full(n + 1), full(n + 1), full(1)
        self.pages = full(pages + 3 if page_cap is None else page_cap)
        self.pos, self.slot, self.seq = (full(rows + 2 if row_cap is None else row_cap) for _ in range(3))

    def call(self, ops, in_place=False):
        lens_out = self.lens if in_place else torch.full_like(self.lens, -5)
        count_out = self.count if in_place else torch.full_like(self.count, -5)
        torch.cuda.synchronize()
        ops.kv_tables(self.lens, self.add, self.table, self.free, self.count, lens_out, count_out, self.indptr, self.pages, self.row_ptr,
                      self.pos, self.slot, self.seq, self.status)
        ops.sync()
        return lens_out.tolist(), count_out.item()

    def check(self, lens_out, count_out):
        lens, stack, table, indptr, pages, row_ptr, rows = tables_of(self.lens0, self.add0, self.table0, self.free0, self.spare)
        assert self.status.item() == 0
        assert lens_out == lens and count_out == len(stack)
        assert np.array_equal(self.table.cpu().numpy(), table)
        free = self.free.cpu().numpy()
        assert list(free[:len(stack)]) == stack
        assert self.indptr.tolist() == indptr and self.row_ptr.tolist() == row_ptr
        assert self.pages.tolist() == [int(p) for p in pages] + [-5] * (len(self.pages) - len(pages))
        pad = [(-1, -1, -1)] * (len(self.pos) - len(rows))
        assert list(zip(self.pos.tolist(), self.slot.tolist(), self.seq.tolist())) == [tuple(int(x) for x in r) for r in rows] + pad


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n", [0, 1, 2, 31, 33, 64, 511, 512, 513, 1025, 4096])
def test_tables_of_mixed_requests(ops, n, in_place):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 90, n)
    add = rng.choice([-1, 0, 1, 1, 1, 5, 16, 17, 40], n)
    t = Tables(lens.tolist(), add.tolist(), 9, 3 * n + 2, seed=n)
    t.check(*t.call(ops, in_place))


@pytest.mark.parametrize("lens,add,spare", [
    ([0], [0], 0), ([0], [-1], 0), ([16], [1], 1), ([15], [1], 0), ([0], [1], 1), ([17], [-1], 0),
    ([100, 0], [-1, 112], 0),             # the pages that come back are taken in the same call, all seven
    ([100, 0], [-1, 120], 1),             # and one more
    ([100, 0], [-1, 30], 5),              # fewer than came back
    ([0] * 40, [0] * 40, 3), ([50] * 40, [-1] * 40, 0),
    ([0] * 30 + [20000], [0] * 30 + [3000], 188),  # one long sequence behind empty ones: more rows than a CTA has threads
])
def test_tables_of_edge_requests(ops, lens, add, spare):
    t = Tables(lens, add, 1500, spare)
    t.check(*t.call(ops))


@pytest.mark.parametrize("lens,add,kw,status", [
    ([5, -1], [1, 1], {}, 1), ([5, 5], [1, -2], {}, 1), ([60, 60], [1, 5], {}, 1), ([5, 5], [2**31 - 1, 1], {}, 1), ([2**31 - 1, 5], [2**31 - 1, 1], {}, 1),
    ([16, 16, 16], [1, 1, 1], {"spare": 2}, 2), ([20, 20], [1, 1], {"row_cap": 1}, 4), ([20, 20], [1, 1], {"page_cap": 3}, 8),
    ([40, 5], [-1, 1], {"spare": 2, "free_cap": 4}, 16), ([16, 16], [1, 1], {"spare": 1, "row_cap": 0, "page_cap": 0}, 2 + 4 + 8),
])
def test_tables_refusals_change_nothing(ops, lens, add, kw, status):
    held = [min(max(c, 0), 60) for c in lens]
    t = Tables(held, [0] * len(lens), 4, kw.pop("spare", 8), **{"row_cap": 4, "page_cap": 8, **kw})
    t.lens, t.add = i32(lens), i32(add)
    lens_out, count_out = t.call(ops)
    assert t.status.item() == status
    assert lens_out == lens and count_out == t.spare
    assert np.array_equal(t.table.cpu().numpy(), t.table0) and np.array_equal(t.free.cpu().numpy(), t.free0)
    assert (t.pages == -5).all() and (t.indptr == 0).all() and (t.row_ptr == 0).all()
    assert (t.pos == -1).all() and (t.slot == -1).all() and (t.seq == -1).all()


@pytest.mark.parametrize("count", [-1, 9, 2**31 - 1])
def test_tables_refuse_a_height_outside_the_stack(ops, count):
    t = Tables([5, 5], [1, 1], 4, 8, free_cap=8)
    t.count = i32([count])
    lens_out, count_out = t.call(ops)
    assert t.status.item() & 16 and lens_out == [5, 5] and count_out == count


def test_tables_step_in_a_graph(ops):
    """A captured step that keeps lengths and free pages in place, replayed until the pages run out."""
    t = Tables([3, 30, 0, 47], [1, 1, 1, 1], 20, 9, page_cap=64)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.stream(stream.cuda_stream)
        ops.kv_tables(t.lens, t.add, t.table, t.free, t.count, t.lens, t.count, t.indptr, t.pages, t.row_ptr, t.pos, t.slot, t.seq, t.status)
    ops.stream(0)
    lens, table, stack = list(t.lens0), t.table0, list(t.free0[:t.spare])
    for step in range(60):
        graph.replay()
        torch.cuda.synchronize()
        wanted = sum(c % PAGE == 0 for c in lens)
        if wanted > len(stack):
            assert t.status.item() == 2 and t.lens.tolist() == lens and t.count.item() == len(stack)
            break
        lens, stack, table, indptr, pages, row_ptr, rows = tables_of(lens, [1] * 4, table, np.array(stack, dtype=np.int32), len(stack))
        assert t.status.item() == 0 and t.lens.tolist() == lens and t.count.item() == len(stack)
        assert np.array_equal(t.table.cpu().numpy(), table) and t.pages.tolist()[:len(pages)] == [int(p) for p in pages]
        assert t.slot.tolist()[:4] == [int(r[1]) for r in rows]
    else:
        raise AssertionError("the pages did not run out")


# ---- norm + rotary embedding ---------------------------------------------------------------------------------------------

def rope_of(x, gains, pos, d, eps, theta):
    """x [rows, heads, d] in f64, gains [heads, d] or None."""
    if gains is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gains
    a = pos.astype(np.float64)[:, None, None] * np.power(theta, -2.0 * np.arange(d // 2) / d)
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)


def check_rope(got, x, gains, pos, d, eps, theta):
    want = rope_of(x, gains, pos, d, eps, theta)
    # one rounding to bf16 (2^-8 of the value), and before it f32: the mean of d squares and its root (d + 4 roundings at most, half of
    # them count), three products and a sum, an angle off by 2^-24 of a turn's half and a sine off by two more: (d / 2 + 16) * 2^-24
    # of the pair's size. The last term is bf16's smallest step.
    y = x if gains is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gains
    size = np.hypot(y[..., :d // 2], y[..., d // 2:])
    tol = np.abs(want) * 2.0 ** -8 + np.concatenate([size, size], -1) * ((d / 2 + 16) * 2.0 ** -24 * (1 + 2.0 ** -8)) + 2.0 ** -133
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk,rows", [(1, 1, 1), (16, 8, 3), (5, 1, 130), (3, 2, 1023), (7, 7, 1025), (0, 1, 17), (2, 0, 6)])
def test_qk_norm_rope(ops, hq, hk, rows, d):
    rng = np.random.default_rng(rows)
    heads = hq + hk
    x = bf16(rng.standard_normal((rows, (heads + 1) * d)) * 3)  # a head of V behind them
    q_norm, k_norm = bf16(1 + 0.5 * rng.standard_normal(d)), bf16(1 + 0.5 * rng.standard_normal(d))
    pos = rng.integers(0, 40000, rows).astype(np.int32)
    pos[rng.integers(0, rows)] = 2 ** 31 - 1
    pos[rng.integers(0, rows)] = 0
    out = torch.full((rows, heads * d + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope(x, q_norm, k_norm, i32(pos), hq, hk, d, 1e-6, 1e6, out)
    ops.sync()
    gains = np.concatenate([np.tile(f64(q_norm), (hq, 1)), np.tile(f64(k_norm), (hk, 1))])
    xs = f64(x)[:, :heads * d].reshape(rows, heads, d)
    check_rope(f64(out)[:, :heads * d].reshape(rows, heads, d), xs, gains, pos, d, 1e-6, 1e6)
    assert (out[:, heads * d:] == 3).all()


@pytest.mark.parametrize("d", [64, 128])
def test_qk_norm_rope_in_place_skips_rows_and_norms(ops, d):
    rng = np.random.default_rng(d)
    hq, hk, rows = 4, 2, 37
    x = bf16(rng.standard_normal((rows, (hq + 2 * hk) * d)))
    pos = rng.integers(-1, 3, rows).astype(np.int32)
    pos[5] = -2 ** 31
    before = f64(x)
    gain = bf16(1 + 0.5 * rng.standard_normal(d))
    ops.qk_norm_rope(x, None, gain, i32(pos), hq, hk, d, 1e-5, 1e4, x)  # q is rotated as it is
    ops.sync()
    got, live = f64(x), pos >= 0
    assert np.array_equal(got[~live], before[~live]) and np.array_equal(got[:, (hq + hk) * d:], before[:, (hq + hk) * d:])
    xs = before[live].reshape(-1, hq + 2 * hk, d)
    ys = got[live].reshape(-1, hq + 2 * hk, d)
    check_rope(ys[:, :hq], xs[:, :hq], None, pos[live], d, 1e-5, 1e4)
    check_rope(ys[:, hq:hq + hk], xs[:, hq:hq + hk], np.tile(f64(gain), (hk, 1)), pos[live], d, 1e-5, 1e4)


# ---- append ----------------------------------------------------------------------------------------------------------------

def e4m3(x):
    """The nearest E4M3 value, ties to even, at most 448 in magnitude; a NaN stays one."""
    mag = np.where(np.isfinite(x), np.abs(x), 448.0)
    _, e = np.frexp(np.where(mag == 0, 1.0, mag))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    y = np.copysign(np.minimum(np.rint(mag / step) * step, 448.0), x)
    return np.where(np.isnan(x), np.nan, y)


def append_of(kv, scales, k, v, slots):
    """kv [pages, heads, 2, 16, d] as values of codes, scales; both changed in place. Rows run by run."""
    heads, d = kv.shape[1], kv.shape[-1]
    x = np.stack([k.reshape(-1, heads, d), v.reshape(-1, heads, d)], 2)
    r = 0
    while r < len(slots):
        if slots[r] < 0:
            r += 1
            continue
        page, off = divmod(int(slots[r]), PAGE)
        m = 1
        while r + m < len(slots) and off + m < PAGE and slots[r + m] == slots[r] + m:
            m += 1
        for h, w in itertools.product(range(heads), range(2)):
            new = x[r:r + m, h, w]
            top = np.abs(new[np.isfinite(new)]).max(initial=0.0)
            scale = MIN_SCALE
            while top > 448.0 * scale:
                scale *= 2
            if off:
                old = scales[page, h, w]
                scale = max(scale, old)
                if scale > old:
                    kv[page, h, w, :off] = e4m3(kv[page, h, w, :off] * (old / scale))
            kv[page, h, w, off:off + m] = e4m3(new / scale)
            scales[page, h, w] = scale
        r += m


def cache(pages, heads, d, seed, spread=2):
    """A cache with codes of all magnitudes, and NaN codes at some places, as freed pages may hold."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (pages, heads, 2, PAGE, d)).astype(np.uint8)
    scales = np.exp2(rng.integers(-spread, spread + 1, (pages, heads, 2))).astype(np.float32)
    return torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()


def values(kv):
    return kv.view(torch.float8_e4m3fn).cpu().double().numpy()


def run_append(ops, kv, scales, k, v, slots):
    want, want_scales = values(kv), f64(scales)
    append_of(want, want_scales, f64(k), f64(v), slots)
    ops.kv8_append(k, v, i32(slots), kv, scales)
    ops.sync()
    assert np.array_equal(f64(scales), want_scales)
    got = values(kv)
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:5]
    assert np.array_equal(np.signbit(got) | np.isnan(got), np.signbit(want) | np.isnan(want))


def slots_of(rng, spans, pages):
    """Slots of sequences that hold `c` tokens and get `a` more, over pages of a random order."""
    order = list(rng.permutation(pages))
    slots = []
    for c, a in spans:
        at = [order.pop() for _ in range(-(-(c + a) // PAGE))]
        slots += [at[p // PAGE] * PAGE + p % PAGE for p in range(c, c + a)]
    return slots


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,spans", [
    (1, [(0, 1)]), (2, [(7, 1)]), (3, [(15, 1), (16, 1)]), (1, [(0, 16)]), (2, [(0, 17)]), (2, [(5, 30)]), (1, [(15, 33)]),
    (2, [(i, 1) for i in range(40)]), (2, [(3, 13), (0, 31), (9, 7), (1, 15), (14, 2), (0, 48), (15, 1)]), (8, [(0, 100), (40, 100)]),
])
def test_append_matches_the_definition(ops, heads, spans, d):
    rng = np.random.default_rng(len(spans))
    pages = sum(-(-(c + a) // PAGE) for c, a in spans) + 2
    kv, scales = cache(pages, heads, d, len(spans))
    slots = slots_of(rng, spans, pages)
    rows = bf16(rng.standard_normal((len(slots), (2 * heads + 1) * d)) * np.exp2(rng.integers(-12, 13, (len(slots), 1))))
    run_append(ops, kv, scales, rows[:, d:(heads + 1) * d], rows[:, (heads + 1) * d:], slots)


@pytest.mark.parametrize("d", [64, 128])
def test_append_skips_rows_without_a_slot(ops, d):
    """A padded batch: rows without a slot in front of, between and behind the sequences' rows."""
    rng = np.random.default_rng(3)
    spans = [(0, 9), (4, 30), (2, 1), (15, 2)]
    at = slots_of(rng, spans, 9)
    slots = [-1]
    for _, a in spans:
        slots += at[:a] + [-1, -5]
        at = at[a:]
    kv, scales = cache(9, 2, d, 3)
    k, v = bf16(rng.standard_normal((len(slots), 2 * d))), bf16(rng.standard_normal((len(slots), 2 * d)))
    run_append(ops, kv, scales, k, v, slots)


@pytest.mark.parametrize("d", [64, 128])
def test_append_of_special_values(ops, d):
    """Zeros, the largest and the smallest numbers, infinities and NaN; borders of a scale; a page whose scale jumps."""
    heads, pages = 2, 12
    tops = [0.0, 3.3895313892515355e38, 1e-38, 9.2e-41, 448.0, 450.0, 224.0, 2.0 ** -100, 448 * 2.0 ** -100, 449 * 2.0 ** -100, 1.75, 1.7578125]
    rng = np.random.default_rng(5)
    for c in (0, 5, 15):
        kv, scales = cache(pages, heads, d, c)
        x = rng.uniform(-1, 1, (pages, 2 * heads * d)) * np.array(tops)[:, None]
        x[:, ::7] = np.array(tops)[:, None]
        x[1::2, 3], x[2::3, 5], x[::4, 9] = np.inf, -np.inf, np.nan
        x[3, :d] = np.nan  # a head of nothing else
        x[4, :d] = np.inf
        rows = bf16(x)
        run_append(ops, kv, scales, rows[:, :heads * d], rows[:, heads * d:], [p * PAGE + c for p in range(pages)])


def test_append_token_by_token_keeps_what_it_can(ops):
    """A page that is filled one token at a time: codes within half a step of the final scale of what was put in, or of the step
    they had under an earlier scale."""
    heads, d = 2, 128
    rng = np.random.default_rng(8)
    kv, scales = cache(2, heads, d, 9)
    x = rng.standard_normal((PAGE, 2 * heads * d)) * np.exp2(np.linspace(-3, 6, PAGE))[:, None]
    rows = bf16(x)
    for i in range(PAGE):
        run_append(ops, kv, scales, rows[i:i + 1, :heads * d], rows[i:i + 1, heads * d:], [PAGE + i])
    got = values(kv)[1] * f64(scales)[1][..., None, None]
    want = np.stack([f64(rows)[:, :heads * d].reshape(PAGE, heads, d), f64(rows)[:, heads * d:].reshape(PAGE, heads, d)], 2).transpose(1, 2, 0, 3)
    # e4m3: 2^-4 of the value, and half a step of the smallest numbers of the final scale for each of at most 9 doublings
    tol = np.abs(want) * 2.0 ** -4 * (1 + 2.0 ** -4) + f64(scales)[1][..., None, None] * 2.0 ** -10 * 2
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("bad", [9 * PAGE, 2 ** 31 - 1])
def test_append_outside_the_cache_is_reported(ops, bad):
    from pega_omni_b200.ops import OpsError
    kv, scales = cache(9, 2, 64, 1)
    before, scales_before = kv.clone(), scales.clone()
    k = bf16(np.ones((1, 128)))
    ops.kv8_append(k, k, i32([bad]), kv, scales)
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()
    assert torch.equal(kv, before) and torch.equal(scales, scales_before)


@pytest.mark.parametrize("front", [0, 13, 15, 31])
@pytest.mark.parametrize("given,out", [
    ([0, 0, 1, 2, 20, 20, 20, 37, 36, 50, 53, 64, 65, 64], {1, 5, 6, 8, 10, 13}),
    ([638, 638, 639], {1}), ([637, 639, 638], {1, 2}),  # at the end of the last page
    ([0] + list(range(16)), {1}),
])
def test_append_leaves_out_rows_that_are_not_their_pages_next(ops, front, given, out):
    """The same slot twice, slots that descend or skip one, behind one another and where the kernel changes warps."""
    from pega_omni_b200.ops import OpsError
    given = [16 * (i + 6) for i in range(front)] + given
    kept = [i for i in range(len(given)) if i - front not in out]
    rng = np.random.default_rng(front)
    kv, scales = cache(40, 2, 64, 2)
    k, v = bf16(rng.standard_normal((len(given), 128))), bf16(rng.standard_normal((len(given), 128)))
    want, want_scales = values(kv), f64(scales)
    append_of(want, want_scales, f64(k)[kept], f64(v)[kept], [given[i] for i in kept])
    ops.kv8_append(k, v, i32(given), kv, scales)
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()
    assert np.array_equal(f64(scales), want_scales) and np.array_equal(values(kv), want, equal_nan=True)


# ---- attention over the pages ---------------------------------------------------------------------------------------------

def attend_case(hq, hk, d, lens, seed, spread=2, extra=3, loud=1.0):
    rng = np.random.default_rng(seed)
    counts = [-(-t // PAGE) for t in lens]
    kv, scales = cache(sum(counts) + extra, hk, d, seed, spread)
    order = rng.permutation(sum(counts) + extra).astype(np.int32)
    indptr = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    # tokens that are attended to hold numbers; behind a sequence's end and in pages of nobody NaN codes stay
    codes = kv.cpu().numpy()
    for s, t in enumerate(lens):
        for i in range(counts[s]):
            page = order[indptr[s] + i]
            m = min(PAGE, t - i * PAGE)
            part = codes[page, :, :, :m]
            codes[page, :, :, :m] = np.where((part & 0x7f) >= 0x78, part & 0x80 | 0x38 | part & 7, part)  # at most 240
            codes[page, :, :, m:] = 0x7f
    q = bf16(rng.standard_normal((len(lens), hq * d)) * loud / 100)
    return torch.from_numpy(codes).cuda(), scales, order[:sum(counts)], indptr, q


def attend_of(q, kv, scales, pages, indptr, lens, hq, hk, d, scale):
    """(result, its tolerance) in f64."""
    out, tol = np.zeros((len(lens), hq * d)), np.zeros((len(lens), hq * d))
    vals, scales, q = values(kv), f64(scales), f64(q)
    for n, t in enumerate(lens):
        if t <= 0:
            continue
        at = pages[indptr[n]:indptr[n] + -(-t // PAGE)]
        x = (vals[at] * scales[at][..., None, None]).transpose(1, 2, 0, 3, 4).reshape(hk, 2, -1, d)[:, :, :t]
        for h in range(hq):
            k, v = x[h // (hq // hk)]
            qh = q[n, h * d:(h + 1) * d]
            s = k @ qh * scale
            w = np.exp(s - s.max())
            l = w.sum()
            w /= l
            o, a = w @ v, w @ np.abs(v)
            # the result's rounding (2^-8); the weights' rounding to f16 (2^-11, or 2^-25 of the largest weight, of which the reference
            # is at most a factor of 1 away); their exponent: a score is a sum of d products, each addition off by 2^-23 of the
            # magnitudes at most, and scaled by products of f32 (another 4); ex2 and the f32 sums over t tokens (t / 2 + 8 roundings)
            ds = (d + 4) * 2.0 ** -23 * (np.abs(k) @ np.abs(qh)).max() * abs(scale)
            r = 2.0 ** -11 + 2 * ds + (t / 2 + 8) * 2.0 ** -23
            out[n, h * d:(h + 1) * d] = o
            tol[n, h * d:(h + 1) * d] = np.abs(o) * 2.0 ** -8 + (a * r + np.abs(v).max() * t * 2.0 ** -25 * w.max()) * (1 + 2.0 ** -7) + 1e-38
    return out, tol


def run_attend(ops, q, kv, scales, pages, indptr, lens, hq, hk, d, scale, seq=None, pos=None):
    out = torch.full((len(lens), hq * d + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q, kv, scales, i32([t - 1 for t in lens] if pos is None else pos), i32(indptr), i32(pages), hq, scale, out[:, :hq * d],
                   None if seq is None else i32(seq))
    ops.sync()
    assert (out[:, hq * d:] == 3).all()
    return f64(out[:, :hq * d])


def check_attend(ops, hq, hk, d, lens, seed=0, scale=None, **kw):
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, seed, **kw)
    scale = d ** -0.5 if scale is None else scale
    want, tol = attend_of(q, kv, scales, pages, indptr, lens, hq, hk, d, scale)
    got = run_attend(ops, q, kv, scales, pages, indptr, lens, hq, hk, d, scale)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / np.maximum(tol, 1e-30)).max()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [0], [16], [17], [0, 1, 2, 15, 16, 17, 31, 33, 0], [127, 128, 129, 130], [1023, 4100, 5], [1] * 33])
def test_attend_lengths(ops, lens, d):
    check_attend(ops, 4, 2, d, lens, seed=len(lens))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (2, 1), (15, 3), (7, 1), (8, 1), (18, 2), (16, 1), (17, 1), (33, 1), (80, 2), (16, 8), (32, 8)])
def test_attend_head_groups(ops, hq, hk, d):
    check_attend(ops, hq, hk, d, [70, 3, 0, 300], seed=hq)


@pytest.mark.parametrize("rows", [1, 3, 20, 100, 300])
def test_attend_every_split(ops, rows):
    """From rows that a cluster shares to rows that have one CTA each."""
    rng = np.random.default_rng(rows)
    check_attend(ops, 4, 2, 128, rng.integers(0, 700, rows).tolist(), seed=rows)


@pytest.mark.parametrize("hq,hk,d,lens", [
    (2, 1, 128, [5000]), (9, 1, 64, [4096, 4097]), (17, 1, 128, [9000, 0, 3]), (6, 3, 64, [0, 12001, 1, 0, 700]), (5, 1, 128, [40000]),
    (4, 4, 64, [6000, 5999, 16, 8192]), (16, 8, 128, [4500, 4111]),
])
def test_attend_long_rows_in_pieces(ops, hq, hk, d, lens):
    """Few rows of many tokens, which are cut into pieces and joined; short and empty rows between them."""
    check_attend(ops, hq, hk, d, lens, seed=hq + len(lens), loud=3.0)


def test_attend_pieces_of_rows_that_are_wrong(ops):
    """A long row that ends outside its pages is reported and becomes zeros; a page outside the cache is left out; the others stand."""
    from pega_omni_b200.ops import OpsError
    hq, hk, d, lens = 4, 2, 64, [9000, 5000, 7000]
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, 61)
    want, tol = attend_of(q, kv, scales, pages, indptr, lens, hq, hk, d, 0.1)
    pages[int(indptr[1]) + 200] = kv.shape[0]
    out = torch.full((3, hq * d), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q, kv, scales, i32([9010, 4999, 6999]), i32(indptr), i32(pages), hq, 0.1, out)
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()
    got = f64(out)
    assert (got[0] == 0).all() and np.isfinite(got[1]).all() and (np.abs(got[2] - want[2]) <= tol[2]).all()


@pytest.mark.parametrize("loud", [0.01, 10.0, 100.0])
@pytest.mark.parametrize("spread", [0, 8])
def test_attend_flat_and_peaked(ops, loud, spread):
    """Nearly equal weights, and rows that one token has almost to itself; page scales far apart."""
    check_attend(ops, 6, 2, 64, [1, 500, 37, 1000], seed=3, loud=loud, spread=spread)
    check_attend(ops, 6, 2, 128, [1, 500, 37, 1000], seed=4, loud=loud, spread=spread)


def test_attend_scales_apart_by_much(ops):
    """Pages whose V scales are 2^60 apart, the loud ones with small weights and the other way round; scales that are no powers of
    two, and zero."""
    hq, hk, d, lens = 4, 1, 128, [64, 64]
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, 11, loud=3.0)
    rng = np.random.default_rng(1)
    scales = torch.from_numpy((rng.uniform(1, 2, tuple(scales.shape)) / 64).astype(np.float32)).cuda()
    scales[int(pages[1]), :, 1] = 2.0 ** 30 * 1.5
    scales[int(pages[2]), :, 1] = 2.0 ** -30
    scales[int(pages[5]), :, 1] = 0
    scales[int(pages[6]), :, 0] = 0
    scales[int(pages[4]), :, 1] = 2.0 ** -100
    want, tol = attend_of(q, kv, scales, pages, indptr, lens, hq, hk, d, 0.3)
    got = run_attend(ops, q, kv, scales, pages, indptr, lens, hq, hk, d, 0.3)
    assert (np.abs(got - want) <= tol).all()
    scales[:, :, 1] = 0  # nothing but zeros
    assert (run_attend(ops, q, kv, scales, pages, indptr, lens, hq, hk, d, 0.3) == 0).all()


def test_attend_rows_of_one_sequence(ops):
    """Rows that name their sequence: several of one, in any order, rows behind the last without one."""
    hq, hk, d = 8, 4, 64
    kv, scales, pages, indptr, _ = attend_case(hq, hk, d, [90, 0, 40], 21)
    seq, pos = [2, 0, 0, 2, 0, -1, 1], [39, 89, 4, 0, 89, -1, -1]
    q = bf16(np.random.default_rng(2).standard_normal((7, hq * d)) / 50)
    full = [int(indptr[s]) if s >= 0 else 0 for s in seq]
    want, tol = np.zeros((7, hq * d)), np.zeros((7, hq * d))
    for n, (s, p) in enumerate(zip(seq, pos)):
        want[n], tol[n] = (x[0] for x in attend_of(q[n:n + 1], kv, scales, pages, np.array([full[n], full[n]]), [p + 1], hq, hk, d, 0.2))
    got = run_attend(ops, q, kv, scales, pages, indptr, [p + 1 for p in pos], hq, hk, d, 0.2, seq=seq, pos=pos)
    assert (np.abs(got - want) <= tol).all() and (got[5:] == 0).all()


def test_attend_is_the_same_every_time(ops):
    kv, scales, pages, indptr, q = attend_case(16, 8, 128, [900, 20, 1700], 31)
    runs = [run_attend(ops, q, kv, scales, pages, indptr, [900, 20, 1700], 16, 8, 128, 0.1) for _ in range(3)]
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


def test_attend_not_a_number(ops):
    """A NaN among a row's own tokens or queries reaches that row and no other."""
    hq, hk, d, lens = 2, 1, 128, [40, 40, 40]
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, 41)
    kv[int(pages[indptr[1] + 2]), 0, 0, 7, 3] = 0x7f   # the last key of row 1
    q[2, 5] = float("nan")                              # head 0 of row 2
    want, tol = attend_of(q, kv, scales, pages, indptr, [40, 0, 40], hq, hk, d, 0.1)
    got = run_attend(ops, q, kv, scales, pages, indptr, lens, hq, hk, d, 0.1)
    assert np.isnan(got[1]).all() and np.isnan(got[2, :d]).all()
    for part in (np.s_[0], np.s_[2, d:]):
        assert (np.abs(got[part] - want[part]) <= tol[part]).all()


@pytest.mark.parametrize("lens", [[40], [700], [9000], [300, 9000], [600] * 300])
def test_attend_scores_without_bound(ops, lens):
    """Infinities in a query: the softmax of that head is no number, however the row is cut, and nothing else notices."""
    hq, hk, d = 2, 1, 128
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, 43)
    want, tol = attend_of(q, kv, scales, pages, indptr, lens, hq, hk, d, 0.1)
    q[len(lens) - 1, 7] = float("inf")
    out = torch.full((len(lens), hq * d), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q, kv, scales, i32([t - 1 for t in lens]), i32(indptr), i32(pages), hq, 0.1, out)
    ops.sync()
    got = f64(out)
    assert np.isnan(got[-1, :d]).all()
    assert (np.abs(got[:-1] - want[:-1]) <= tol[:-1]).all() and (np.abs(got[-1, d:] - want[-1, d:]) <= tol[-1, d:]).all()


@pytest.mark.parametrize("what", ["page", "negative page", "sequence", "range", "count"])
def test_attend_outside_its_tables_is_reported(ops, what):
    from pega_omni_b200.ops import OpsError
    hq, hk, d, lens = 4, 2, 64, [40, 20]
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, 51)
    want, tol = attend_of(q, kv, scales, pages, indptr, lens, hq, hk, d, 0.1)
    seq, pos = [0, 1], [39, 19]
    if what.endswith("page"):
        pages[1] = kv.shape[0] if what == "page" else -3
    elif what == "sequence":
        seq[0] = 2
    elif what == "range":
        indptr[0] = -4
    else:
        pos[0] = 48  # a fourth page, which the sequence does not have
    out = torch.full((2, hq * d), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q, kv, scales, i32(pos), i32(indptr), i32(pages), hq, 0.1, out, i32(seq))
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()
    got = f64(out)
    assert (np.abs(got[1] - want[1]) <= tol[1]).all()
    assert np.isfinite(got[0]).all() and (what.endswith("page") or (got[0] == 0).all())


@pytest.mark.parametrize("hq,hk,d,length", [(4, 2, 64, 9), (16, 1, 128, 700), (4, 2, 128, 9000)])
def test_attend_without_any_page_is_zero(ops, hq, hk, d, length):
    """All of a row's pages outside the cache: nothing is left to attend to; the other row does not notice."""
    from pega_omni_b200.ops import OpsError
    lens = [length, length]
    kv, scales, pages, indptr, q = attend_case(hq, hk, d, lens, 77)
    want = run_attend(ops, q, kv, scales, pages, indptr, lens, hq, hk, d, 0.1)
    pages = pages.copy()
    pages[:indptr[1]] = -3
    out = torch.full((2, hq * d), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q, kv, scales, i32([t - 1 for t in lens]), i32(indptr), i32(pages), hq, 0.1, out)
    with pytest.raises(OpsError, match="0x2"):
        ops.sync()
    assert (out[0] == 0).all() and np.array_equal(f64(out)[1], want[1])


def test_attend_and_append_far_into_a_large_cache(ops):
    """Pages whose byte offsets pass 32 bits."""
    hq, hk, d = 4, 2, 128
    total = 1 << 20  # 8 GiB
    kv = torch.empty((total, hk, 2, PAGE, d), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((total, hk, 2), device="cuda")
    rng = np.random.default_rng(6)
    pages = np.array([total - 1, 600001, 524289], dtype=np.int32)
    rows = bf16(rng.standard_normal((41, 2 * hk * d)))
    slots = [int(pages[p // PAGE]) * PAGE + p % PAGE for p in range(41)]
    ops.kv8_append(rows[:, :hk * d], rows[:, hk * d:], i32(slots), kv, scales)
    q = bf16(rng.standard_normal((1, hq * d)))
    got = run_attend(ops, q, kv, scales, pages, np.array([0, 3], dtype=np.int32), [41], hq, hk, d, 0.1)
    at = torch.from_numpy(pages.astype(np.int64)).cuda()
    want, tol = attend_of(q, kv[at].contiguous(), scales[at], np.arange(3), np.array([0, 3]), [41], hq, hk, d, 0.1)
    assert (np.abs(got - want) <= tol).all()


def test_calls_on_two_streams_and_from_graphs(ops):
    """No two calls share memory: graphs of one context replayed side by side give what each gives by itself."""
    hq, hk, d = 16, 8, 128
    cases = [attend_case(hq, hk, d, lens, 60 + i) + (lens,) for i, lens in enumerate(([700, 9, 2000], [1500, 1, 64, 333], [9000, 4000], [7000]))]
    want = [run_attend(ops, q, kv, sc, pages, indptr, lens, hq, hk, d, 0.1) for kv, sc, pages, indptr, q, lens in cases]
    held, graphs, streams, outs = [], [], [], []
    for kv, sc, pages, indptr, q, lens in cases:
        held.append((i32([t - 1 for t in lens]), i32(indptr), i32(pages)))
        outs.append(torch.zeros((len(lens), hq * d), dtype=torch.bfloat16, device="cuda"))
        streams.append(torch.cuda.Stream())
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1], stream=streams[-1]):
            ops.stream(streams[-1].cuda_stream)
            ops.kv8_attend(q, kv, sc, *held[-1], hq, 0.1, outs[-1])
        ops.stream(0)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert np.array_equal(f64(o), w)
    ops.sync()


def test_a_stream_of_the_caller(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    s = torch.cuda.Stream()
    kv, scales, pages, indptr, q = attend_case(4, 2, 64, [50], 71)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        o.stream(s.cuda_stream)
        out = torch.empty((1, 4 * 64), dtype=torch.bfloat16, device="cuda")
        o.kv8_attend(q, kv, scales, i32([49]), i32(indptr), i32(pages), 4, 0.1, out)
        doubled = out.float() * 2  # ordered behind the call
    s.synchronize()
    want, tol = attend_of(q, kv, scales, pages, indptr, [50], 4, 2, 64, 0.1)
    assert (np.abs(f64(doubled) / 2 - want) <= tol).all()
    o.stream()
    o.kv8_attend(q, kv, scales, i32([49]), i32(indptr), i32(pages), 4, 0.1, out)
    torch.cuda.synchronize()
    o.sync()
    assert (np.abs(f64(out) - want) <= tol).all()
    o.close()
