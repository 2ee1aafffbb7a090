"""What the calls over a cache of 8 bits refuse on the host, before any device
work (CPU)."""
import ctypes as C

import pytest
import torch


def _lib():
    from ghostflow_hip import _lib as L
    return L, L.load()


def _kv(L, **kw):
    # addresses that are never read: every call below fails first, or is empty
    f = dict(k_pages=16, v_pages=16, dtype=L.U8, num_pages=8, page_size=16, kv_heads=2, head_dim=64,
             page_stride=16 * 2 * 64, row_stride=2 * 64, head_stride=64, page_table=16, max_pages=4, table_stride=4,
             num_seqs=1, kv_lens=16, q_offsets=16, status=None)
    f.update(kw)
    return L.PagedKv(**f)


def _scales(L, **kw):
    f = dict(k=16, v=16, page_stride=32, head_stride=16)
    f.update(kw)
    return L.PagedScales(**f)


def _ref(x):
    return None if x is None else C.byref(x)


def _attend(lib, kv, scales, dtype, tokens=1, heads=4, ldq=256, scale=1.0, window=0, ws=None):
    return lib.gfh_paged_attention_q8(_ref(kv), _ref(scales), dtype, tokens, heads, 16, ldq, 16, 256, scale, 1, window, 0,
                                      ws, 0, None)


def _append(lib, kv, scales, dtype, tokens=1, heads=4, q=16, qo=16, qn=None, kn=None, eps=1e-6, cos=None, rot=0, rows=0):
    return lib.gfh_paged_append_norm(_ref(kv), _ref(scales), dtype, tokens, heads, q, 256, qo, 256, 16, 128, 16, 128, cos,
                                     cos, rows, rot, 0, qn, kn, eps, None)


def _read(lib, kv, scales, dtype, tokens=1, heads=4, ldk=128):
    return lib.gfh_paged_read(_ref(kv), _ref(scales), dtype, tokens, 16, ldk, 16, 128, None)


CALLS = (_attend, _append, _read)


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=8), b"multiple of 16"), (dict(head_dim=72), b"multiple of 16"), (dict(head_dim=144), b"head_dim"),
    (dict(kv_heads=0), b"kv_heads"), (dict(page_size=0), b"page_size"), (dict(max_pages=2 ** 29), b"max_pages"),
    (dict(table_stride=3), b"table_stride"), (dict(page_stride=24), b"16-byte"), (dict(row_stride=8), b"16-byte"),
    (dict(head_stride=-16), b"16-byte"), (dict(num_pages=2 ** 30, page_stride=2 ** 40), b"overflows"),
])
def test_shapes(change, word):
    L, lib = _lib()
    for f in CALLS:
        assert f(lib, _kv(L, **change), _scales(L), L.BF16) == L.INVALID_SHAPE
        assert word in lib.gfh_last_error(), lib.gfh_last_error()


def test_types_go_together():
    L, lib = _lib()
    for f in CALLS:
        for kv, s, dt in ((L.BF16, _scales(L), L.BF16), (L.U8, _scales(L), L.U8), (L.U8, _scales(L), 5)):
            assert f(lib, _kv(L, dtype=kv), s, dt) == L.INVALID_DATA
            assert b"dtype" in lib.gfh_last_error()
    # without scales: not over codes, and the float caches' own rule
    for f in (_append, _read):
        assert f(lib, _kv(L), None, L.BF16) == L.INVALID_DATA
    assert _attend(lib, _kv(L), None, L.BF16) == L.NULL_POINTER
    assert _append(lib, _kv(L, dtype=L.F16), None, L.BF16) == L.INVALID_DATA
    assert lib.gfh_paged_attention(C.byref(_kv(L)), L.BF16, 1, 4, 16, 256, 16, 256, 1.0, 1, 0, 0, None, 0,
                                   None) == L.INVALID_DATA


def test_scales():
    L, lib = _lib()
    for f in CALLS:
        for kw in (dict(page_stride=-1), dict(head_stride=-1)):
            assert f(lib, _kv(L), _scales(L, **kw), L.F32) == L.INVALID_SHAPE
            assert b"scales" in lib.gfh_last_error()


def test_calls():
    L, lib = _lib()
    kv, s = _kv(L), _scales(L)
    for f in CALLS:
        assert f(lib, None, s, L.BF16) == L.NULL_POINTER
        assert f(lib, kv, s, L.BF16, tokens=-1) == L.INVALID_SHAPE
        assert f(lib, kv, s, L.BF16, tokens=0) == 0
        assert f(lib, _kv(L, num_seqs=0), s, L.BF16) == 0
        # host memory
        assert f(lib, kv, s, L.BF16) in (L.INVALID_DATA, L.COMPUTATION_FAILED)
    assert _attend(lib, kv, s, L.BF16, window=-1) == L.INVALID_SHAPE
    for scale in (float("nan"), float("inf"), 3e38):
        assert _attend(lib, kv, s, L.BF16, scale=scale) == L.INVALID_DATA
    assert _append(lib, kv, s, L.BF16, qo=None) == L.NULL_POINTER
    assert _append(lib, kv, s, L.BF16, q=None, qo=None, qn=16) == L.NULL_POINTER
    for eps in (-1e-6, float("nan"), float("inf")):
        assert _append(lib, kv, s, L.BF16, kn=16, eps=eps) == L.INVALID_DATA
        assert b"norm_eps" in lib.gfh_last_error()
    assert _append(lib, kv, s, L.BF16, cos=16, rot=20, rows=64) == L.INVALID_SHAPE
    assert _append(lib, kv, s, L.BF16, cos=16, rot=64, rows=63) == L.INVALID_SHAPE


def test_more_tokens_than_a_launch_can_have():
    L, lib = _lib()
    kv, s = _kv(L, head_dim=16, kv_heads=1), _scales(L)
    most = 4 * (2 ** 24 - 1)
    for tokens in (most, most + 1, 2 ** 30):
        rc = lib.gfh_paged_read(C.byref(kv), C.byref(s), L.BF16, tokens, 16, 16, 16, 16, None)
        assert (rc == L.INVALID_SHAPE) == (tokens > most)
        rc = lib.gfh_paged_append_norm(C.byref(kv), C.byref(s), L.BF16, tokens, 1, 16, 16, 16, 16, 16, 16, 16, 16, None, None,
                                       0, 0, 0, None, None, 0.0, None)
        assert (rc == L.INVALID_SHAPE) == (tokens > most)


def test_workspace_size():
    L, lib = _lib()
    size = lib.gfh_paged_attention_q8_workspace_size
    assert size(C.byref(_kv(L, head_dim=8)), 1, 4, 0, 0) == 0
    assert size(C.byref(_kv(L, dtype=L.BF16)), 1, 4, 0, 0) == 0
    assert size(C.byref(_kv(L)), 0, 4, 0, 0) == 0
    long = _kv(L, max_pages=4096, table_stride=4096)
    few, most = size(C.byref(long), 1, 4, 0, 4000), size(C.byref(long), 1, 4, 0, 0)
    assert 0 < few < most and most % 4 == 0


def test_packed_struct():
    L, _ = _lib()
    from ghostflow_hip import ops
    s = L.PagedScales.from_buffer_copy(ops._PAGED_SCALES.pack(1, 2, 3, 4))
    assert [getattr(s, f) for f, _ in L.PagedScales._fields_] == [1, 2, 3, 4]


def test_python_checks():
    import ghostflow_hip as gh
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.uint8)
    steps = torch.zeros(4, 2, 16, dtype=torch.uint8)
    i, off = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    check = gh.ops._paged_scales
    assert check(steps, steps, pages) is not None and check(None, None, pages.float()) is None
    for k, v, p in ((None, None, pages), (steps, None, pages), (steps, steps, pages.float()),
                    (steps[:3], steps[:3], pages), (steps.transpose(1, 2), steps.transpose(1, 2), pages),
                    (steps.float(), steps.float(), pages), (steps, steps.transpose(1, 2).contiguous().transpose(1, 2), pages)):
        with pytest.raises(gh.GhostFlowError):
            check(k, v, p)
    with pytest.raises(gh.GhostFlowError):  # not on a GPU
        gh.paged_read(pages, pages, i[None], off, i, tokens=0, k_scales=steps, v_scales=steps)


def test_cache_of_8_bits():
    import ghostflow_hip as gh
    c = gh.PagedKVCache(6, 4, 2, 16, dtype=torch.uint8, device="cpu")
    assert c.k_pages.dtype == torch.uint8 and c.k_scales.shape == c.v_scales.shape == (6, 2, 4)
    assert gh.PagedKVCache(6, 4, 2, 16, device="cpu").k_scales is None
    with pytest.raises(gh.GhostFlowError):
        c.read(3)
