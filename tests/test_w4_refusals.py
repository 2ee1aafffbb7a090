"""What the 4-bit weight calls refuse on the host (CPU)."""
import pytest


def _lib():
    from ghostflow_hip import _lib as L
    return L, L.load()


def _linear(lib, dtype=2, ldx=64, ldy=8, m=1, n=8, k=64, group=32, codes=16, ws=None):
    return lib.gfh_linear_w4(dtype, 16, ldx, codes, 16, None, None, 16, ldy, m, n, k, group, ws, 0, None)


@pytest.mark.parametrize("change,word", [
    (dict(k=48), b"multiple of 32"), (dict(k=-32), b"out of range"), (dict(n=-1), b"out of range"),
    (dict(group=16), b"group"), (dict(group=48), b"group"), (dict(group=0), b"group"), (dict(m=-1), b"m=-1"),
    (dict(m=2 ** 20), b"out of range"), (dict(ldx=63), b"ldx"), (dict(ldy=7), b"ldy"), (dict(k=0, ldx=0), b"columns"),
])
def test_linear(change, word):
    L, lib = _lib()
    assert _linear(lib, **change) == L.INVALID_SHAPE
    assert word in lib.gfh_last_error(), lib.gfh_last_error()


def test_linear_type_and_nothing_to_do():
    L, lib = _lib()
    assert _linear(lib, dtype=5) == L.INVALID_DATA
    assert _linear(lib, m=0) == 0
    assert _linear(lib, n=0, ldy=0) == 0
    assert _linear(lib) in (L.INVALID_DATA, L.COMPUTATION_FAILED)  # host memory


@pytest.mark.parametrize("n,k,group", [(4, 40, 32), (4, 64, 8), (4, 64, -32), (-1, 64, 32)])
def test_quantize(n, k, group):
    L, lib = _lib()
    assert lib.gfh_quantize_i4_grouped(16, n, k, group, 16, 16, None, None) == L.INVALID_SHAPE
    assert lib.gfh_dequantize_i4_grouped(16, 16, None, n, k, group, 16, None) == L.INVALID_SHAPE


def test_empty_and_null():
    L, lib = _lib()
    assert lib.gfh_quantize_i4_grouped(None, 0, 64, 32, None, None, None, None) == 0
    assert lib.gfh_quantize_i4_grouped(None, 4, 64, 32, None, None, None, None) == L.NULL_POINTER
    assert lib.gfh_dequantize_i4_grouped(None, None, None, 4, 64, 32, None, None) == L.NULL_POINTER


def test_workspace_size():
    L, lib = _lib()
    size = lib.gfh_linear_w4_workspace_size
    assert size(2, 1, 4096, 4096, 128) == 0          # the form for few rows has no parts
    assert size(2, 16, 4096, 4096, 128) % (16 * 4096 * 4) == 0
    assert size(9, 16, 4096, 4096, 128) == 0
    assert size(2, 16, 4096, 40, 128) == 0


def test_python_checks():
    torch = pytest.importorskip("torch")
    import ghostflow_hip as gh
    with pytest.raises(gh.GhostFlowError):
        gh.quantize_grouped_i4(torch.zeros(4, 64))
    with pytest.raises(gh.GhostFlowError):
        gh.linear_w4(torch.zeros(1, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1))


@pytest.mark.parametrize("dtype,m,most", [(0, 1, 4 * (2 ** 24 - 1)), (2, 4, 4 * (2 ** 24 - 1)), (1, 5, 128 * (2 ** 23 - 1)),
                                          (2, 5, 128 * (2 ** 23 - 1))])
def test_more_rows_of_the_weight_than_a_launch_can_have(dtype, m, most):
    """Four rows of W per workgroup of 256 threads, or 128 per one of up to 512:
    fewer than 2^32 work-items."""
    L, lib = _lib()
    for n in (most, most + 1):
        rc = _linear(lib, dtype=dtype, m=m, n=n, ldy=n, k=64)
        if n == most:  # goes on to the memory, which is none
            assert rc in (L.INVALID_DATA, L.COMPUTATION_FAILED) and b"launch" not in lib.gfh_last_error()
        else:
            assert rc == L.INVALID_SHAPE and b"more than one launch" in lib.gfh_last_error(), lib.gfh_last_error()
