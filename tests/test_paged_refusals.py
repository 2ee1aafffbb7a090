"""What gfh_paged_append and gfh_paged_attention refuse on the host, before any
device work (CPU)."""
import ctypes as C

import pytest


def _lib():
    from ghostflow_hip import _lib as L
    return L, L.load()


def _kv(L, **kw):
    # addresses that are never read: every call below fails first, or is empty
    f = dict(k_pages=16, v_pages=16, dtype=L.BF16, num_pages=8, page_size=16, kv_heads=2, head_dim=64,
             page_stride=16 * 2 * 64, row_stride=2 * 64, head_stride=64, page_table=16, max_pages=4, table_stride=4,
             num_seqs=1, kv_lens=16, q_offsets=16, status=None)
    f.update(kw)
    return L.PagedKv(**f)


def _attend(lib, kv, dtype, tokens=1, heads=4, ldq=256, ldo=256, scale=1.0, window=0, q=16, out=16):
    return lib.gfh_paged_attention(None if kv is None else C.byref(kv), dtype, tokens, heads, q, ldq, out, ldo, scale, 1,
                                   window, 0, None, 0, None)


def _append(lib, kv, dtype, tokens=1, heads=4, q=16, qo=16, cos=16, sin=16, rows=64, rot=64):
    return lib.gfh_paged_append(None if kv is None else C.byref(kv), dtype, tokens, heads, q, 256, qo, 256, 16, 128, 16,
                                128, cos, sin, rows, rot, 0, None)


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=4), b"head_dim"), (dict(head_dim=20), b"head_dim"), (dict(head_dim=136), b"head_dim"),
    (dict(kv_heads=3), b"kv_heads"), (dict(kv_heads=0), b"kv_heads"),
    (dict(page_size=0), b"page_size"), (dict(num_pages=-1), b"num_pages"), (dict(max_pages=-1), b"max_pages"),
    (dict(max_pages=2 ** 29, page_size=16), b"max_pages"), (dict(table_stride=3), b"table_stride"),
    (dict(page_stride=12), b"16-byte"), (dict(row_stride=-8), b"16-byte"), (dict(head_stride=65), b"16-byte"),
    (dict(num_seqs=-1), b"num_seqs"), (dict(num_pages=2 ** 30, page_stride=2 ** 40), b"overflows"),
])
def test_shapes(change, word):
    L, lib = _lib()
    for rc in (_attend(lib, _kv(L, **change), L.BF16), _append(lib, _kv(L, **change), L.BF16)):
        assert rc == L.INVALID_SHAPE
        assert word in lib.gfh_last_error(), lib.gfh_last_error()


def test_types():
    L, lib = _lib()
    for act, cache in ((L.BF16, L.F16), (L.F16, L.F32), (L.F32, L.F16), (7, 7), (L.BF16, L.F32)):
        for f in (_attend, _append):
            assert f(lib, _kv(L, dtype=cache), act) == L.INVALID_DATA
            assert b"dtype" in lib.gfh_last_error()


def test_calls():
    L, lib = _lib()
    kv = _kv(L)
    assert _attend(lib, None, L.BF16) == L.NULL_POINTER
    assert _attend(lib, kv, L.BF16, window=-1) == L.INVALID_SHAPE
    assert _attend(lib, kv, L.BF16, scale=float("nan")) == L.INVALID_DATA
    assert _attend(lib, kv, L.BF16, scale=float("inf")) == L.INVALID_DATA
    assert _attend(lib, kv, L.BF16, tokens=-1) == L.INVALID_SHAPE
    assert _attend(lib, kv, L.BF16, tokens=2 ** 29) == L.INVALID_SHAPE
    assert _append(lib, kv, L.BF16, qo=None) == L.NULL_POINTER
    assert _append(lib, kv, L.BF16, sin=None) == L.NULL_POINTER
    assert _append(lib, kv, L.BF16, rot=60) == L.INVALID_SHAPE
    assert _append(lib, kv, L.BF16, rot=128) == L.INVALID_SHAPE
    assert _append(lib, kv, L.BF16, rows=63) == L.INVALID_SHAPE
    assert b"positions" in lib.gfh_last_error()
    # nothing to do
    assert _attend(lib, kv, L.BF16, tokens=0) == 0
    assert _append(lib, _kv(L, num_seqs=0), L.BF16) == 0
    # host memory
    assert _attend(lib, kv, L.BF16) in (L.INVALID_DATA, L.COMPUTATION_FAILED)


def test_workspace_size():
    L, lib = _lib()
    size = lib.gfh_paged_attention_workspace_size
    assert size(C.byref(_kv(L, head_dim=7)), 1, 4, 0, 0) == 0
    assert size(C.byref(_kv(L)), 0, 4, 0, 0) == 0
    long = _kv(L, max_pages=4096, table_stride=4096)
    few, most = size(C.byref(long), 1, 4, 0, 2000), size(C.byref(long), 1, 4, 0, 0)
    assert 0 < few < most and most % 4 == 0


def test_packed_struct():
    """The wrappers pack gfh_paged_kv themselves."""
    L, _ = _lib()
    from ghostflow_hip import ops
    assert ops._PAGED_KV.size == C.sizeof(L.PagedKv)
    values = list(range(1, 18))
    kv = L.PagedKv.from_buffer_copy(ops._PAGED_KV.pack(*values))
    assert [getattr(kv, f) for f, _ in L.PagedKv._fields_] == values


def test_python_checks():
    torch = pytest.importorskip("torch")
    import ghostflow_hip as gh
    q = torch.zeros(1, 4, 64)
    pages = torch.zeros(2, 16, 2, 64)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(gh.GhostFlowError):
        gh.paged_attention(q, pages, pages, i[None], torch.zeros(2, dtype=torch.int32), i)
    with pytest.raises(gh.GhostFlowError):
        gh.paged_append(pages, pages, i[None], torch.zeros(2, dtype=torch.int32), i, q[:, :2], q[:, :2])


def test_more_tokens_than_a_launch_can_have():
    L, lib = _lib()
    kv = _kv(L, head_dim=8, kv_heads=1, page_stride=16 * 8, row_stride=8, head_stride=8)
    # a wave of 64 per token: fewer than 2^32 work-items in all
    most = 4 * (2 ** 24 - 1)
    word = b"more than one launch"
    for tokens in (most, most + 1, 2 ** 30):
        rc = lib.gfh_paged_append(C.byref(kv), L.BF16, tokens, 1, 16, 8, 16, 8, 16, 8, 16, 8, None, None, 0, 0, 0, None)
        if tokens <= most:  # goes on to the memory, which is none
            assert rc in (L.INVALID_DATA, L.COMPUTATION_FAILED) and word not in lib.gfh_last_error()
        else:
            assert rc == L.INVALID_SHAPE and word in lib.gfh_last_error(), lib.gfh_last_error()


@pytest.mark.parametrize("scale", [float("nan"), float("-inf"), 3e38, -3e38])
def test_scales_out_of_range(scale):
    """Times log2 e they have to be finite: 0 times them is 0 then."""
    L, lib = _lib()
    assert _attend(lib, _kv(L), L.BF16, scale=scale) == L.INVALID_DATA
    assert b"scale" in lib.gfh_last_error()
    assert _attend(lib, _kv(L), L.BF16, scale=2e38) in (L.INVALID_DATA, L.COMPUTATION_FAILED)
    assert b"scale" not in lib.gfh_last_error()
