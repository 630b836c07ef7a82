"""Refusals of the operators around the 8-bit paged cache: every argument is checked before any CUDA call, so they are the same
on a machine without a GPU (where the context exists but could not be set up)."""
import ctypes as C

import pytest

INVALID, UNSUPPORTED = -1, -5
AT = C.c_void_p(1 << 20)       # an address that nothing reads: every call here is refused
ODD = C.c_void_p((1 << 20) + 2)
OFF8 = C.c_void_p((1 << 20) + 8)


@pytest.fixture(scope="module")
def call(built_lib):
    h = C.c_void_p()
    built_lib.omni_ops_create(0, C.byref(h))
    assert h

    def go(name, args, **change):
        args = {**args, **change}
        rc = getattr(built_lib, name)(h, *args.values())
        return rc, built_lib.omni_ops_last_error(h).decode()

    yield go
    built_lib.omni_ops_destroy(h)


TABLES = dict(lens=AT, add=AT, n=4, table=AT, width=8, free_pages=AT, free_cap=16, free_count=AT, lens_out=AT, free_count_out=AT,
              indptr=AT, pages=AT, page_cap=32, row_ptr=AT, pos=AT, slot=AT, seq=AT, row_cap=4, status=AT)
ROPE = dict(x=AT, ldx=4096, q_norm=AT, k_norm=AT, pos=AT, rows=3, q_heads=16, kv_heads=8, head_dim=128, eps=1e-6, theta=1e6, out=AT, ldo=4096)
APPEND = dict(k=AT, ldk=1024, v=AT, ldv=1024, slot=AT, rows=3, kv=AT, scales=AT, kv_pages=9, kv_heads=8, head_dim=128)
ATTEND = dict(q=AT, ldq=2048, kv=AT, scales=AT, kv_pages=9, pos=AT, seq=AT, indptr=AT, n_seqs=2, pages=AT, n_pages=9, rows=2, q_heads=16,
              kv_heads=8, head_dim=128, scale=0.1, out=AT, ldo=2048)

PACKED = dict(q=AT, ldq=4096, k=AT, ldk=4096, v=AT, ldv=4096, indptr=AT, n=2, rows=9, q_heads=16, kv_heads=8, head_dim=128, scale=0.1, out=AT, ldo=2048)


@pytest.mark.parametrize("change,status", [
    *[({k: None}, INVALID) for k in ("lens", "add", "table", "free_pages", "free_count", "lens_out", "free_count_out", "indptr", "pages",
                                     "row_ptr", "pos", "slot", "seq", "status")],
    *[({k: -1}, INVALID) for k in ("n", "width", "free_cap", "page_cap", "row_cap")],
    ({"width": 0}, INVALID), ({"n": 4097}, UNSUPPORTED), ({"n": 4096, "width": 16385}, UNSUPPORTED),
])
def test_kv_tables_refuses(call, change, status):
    rc, why = call("omni_op_kv_tables", TABLES, **change)
    assert rc == status and why


@pytest.mark.parametrize("change,status", [
    *[({k: None}, INVALID) for k in ("x", "pos", "out")], *[({k: ODD}, INVALID) for k in ("x", "out", "q_norm", "k_norm")],
    ({"rows": -1}, INVALID), ({"theta": 0.0}, INVALID), ({"theta": float("nan")}, INVALID), ({"ldx": 24 * 128 - 8}, INVALID),
    ({"ldx": 4100}, INVALID), ({"ldo": 4092}, INVALID), ({"ldo": 8192}, INVALID),  # in place with another stride
    ({"head_dim": 96}, UNSUPPORTED), ({"q_heads": 0, "kv_heads": 0}, UNSUPPORTED), ({"q_heads": -1}, UNSUPPORTED),
    ({"q_heads": 65535, "kv_heads": 1}, UNSUPPORTED), ({"rows": 2**31 - 1}, UNSUPPORTED), ({"rows": 2**31 - 1, "q_heads": 1, "kv_heads": 0}, UNSUPPORTED),
    ({"rows": 1 << 22, "q_heads": 60000}, UNSUPPORTED),
])
def test_qk_norm_rope_refuses(call, change, status):
    rc, why = call("omni_op_qk_norm_rope", ROPE, **change)
    assert rc == status and why


@pytest.mark.parametrize("change,status", [
    *[({k: None}, INVALID) for k in ("k", "v", "slot", "kv", "scales")], *[({k: ODD}, INVALID) for k in ("k", "v", "kv", "scales")],
    ({"k": OFF8}, INVALID), ({"kv": OFF8}, INVALID), ({"rows": -1}, INVALID), ({"kv_pages": 0}, INVALID), ({"ldk": 1016}, INVALID),
    ({"ldv": 1028}, INVALID), ({"head_dim": 80}, UNSUPPORTED), ({"kv_heads": 0}, UNSUPPORTED), ({"kv_heads": 65536}, UNSUPPORTED),
    ({"rows": 2**31 - 1}, UNSUPPORTED), ({"rows": 1 << 20, "kv_heads": 60000, "ldk": 60000 * 128, "ldv": 60000 * 128}, UNSUPPORTED),
])
def test_kv8_append_refuses(call, change, status):
    rc, why = call("omni_op_kv8_append", APPEND, **change)
    assert rc == status and why


@pytest.mark.parametrize("change,status", [
    *[({k: None}, INVALID) for k in ("q", "kv", "scales", "pos", "indptr", "pages", "out")], *[({k: ODD}, INVALID) for k in ("q", "kv", "scales", "out")],
    ({"rows": -1}, INVALID), ({"kv_pages": 0}, INVALID), ({"n_seqs": -1}, INVALID), ({"n_pages": -1}, INVALID), ({"ldq": 2040}, INVALID),
    ({"ldo": 2052}, INVALID), ({"q_heads": 12}, UNSUPPORTED), ({"q_heads": 0}, UNSUPPORTED), ({"kv_heads": -8}, UNSUPPORTED), ({"head_dim": 256}, UNSUPPORTED),
    ({"rows": 1 << 24}, UNSUPPORTED),
])
def test_kv8_attend_refuses(call, change, status):
    rc, why = call("omni_op_kv8_attend", ATTEND, **change)
    assert rc == status and why


@pytest.mark.parametrize("change,status", [
    *[({k: None}, INVALID) for k in ("q", "k", "v", "indptr", "out")], *[({k: ODD}, INVALID) for k in ("q", "k", "v", "out")],
    ({"rows": -1}, INVALID), ({"n": -1}, INVALID), ({"ldq": 2040}, INVALID), ({"ldk": 1016}, INVALID), ({"ldv": 1028}, INVALID),
    ({"ldo": 2044}, INVALID), ({"ldq": 1 << 40}, INVALID), ({"q_heads": 9}, UNSUPPORTED), ({"kv_heads": 0}, UNSUPPORTED), ({"head_dim": 96}, UNSUPPORTED),
    ({"scale": -0.1}, INVALID), ({"scale": 0.0}, INVALID), ({"scale": float("nan")}, INVALID), ({"scale": float("inf")}, INVALID), ({"rows": 2**31 - 1, "q_heads": 128}, UNSUPPORTED),
    ({"n": 2**31 - 1}, UNSUPPORTED), ({"n": 16385}, UNSUPPORTED), ({"rows": 2**31 - 1, "q_heads": 1, "kv_heads": 1}, UNSUPPORTED),
])
def test_packed_attend_refuses(call, change, status):
    rc, why = call("omni_op_packed_attend", PACKED, **change)
    assert rc == status and why


def test_null_context_is_refused(built_lib):
    for name, args in (("kv_tables", TABLES), ("qk_norm_rope", ROPE), ("kv8_append", APPEND), ("kv8_attend", ATTEND), ("packed_attend", PACKED)):
        assert getattr(built_lib, "omni_op_" + name)(None, *args.values()) == INVALID
    assert built_lib.omni_ops_stream(None, 1, None) == INVALID


def test_no_rows_is_no_call(call):
    for name, args in (("qk_norm_rope", ROPE), ("kv8_append", APPEND), ("kv8_attend", ATTEND), ("packed_attend", PACKED)):
        assert call("omni_op_" + name, args, rows=0)[0] == 0
    assert call("omni_op_packed_attend", PACKED, n=0)[0] == 0
