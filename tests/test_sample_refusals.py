"""What gfh_sample refuses on the host, before any device work (CPU)."""
import ctypes as C

import pytest
import torch


def _call(dtype=2, logits=16, ld=100, rows=2, vocab=100, u=16, settings=True, tokens=16, workspace=None, **kw):
    from ghostflow_hip import _lib as L
    s = L.Sampling(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    for n, v in kw.items():
        setattr(s, n, v)
    return L.load().gfh_sample(dtype, logits, ld, rows, vocab, u, C.byref(s) if settings else None, tokens, None, workspace,
                               0, None)


def test_refusals():
    from ghostflow_hip import _lib as L
    lib = L.load()
    for kw in (dict(rows=-1), dict(rows=2 ** 20 + 1), dict(vocab=0), dict(vocab=2 ** 19 + 1, ld=2 ** 20), dict(ld=99),
               dict(rows=2 ** 20, vocab=2 ** 19, ld=2 ** 19)):
        assert _call(**kw) == L.INVALID_SHAPE, kw
    for kw in (dict(dtype=3), dict(dtype=8), dict(temperature=float("nan")), dict(top_p=float("nan")),
               dict(min_p=float("nan"))):
        assert _call(**kw) == L.INVALID_DATA, kw
    assert _call(settings=False) == L.NULL_POINTER
    assert _call(rows=0) == 0
    assert _call() in (L.INVALID_DATA, L.COMPUTATION_FAILED)  # host memory
    for kw in (dict(logits=None), dict(u=None), dict(tokens=None)):
        assert _call(**kw) in (L.NULL_POINTER, L.INVALID_DATA, L.COMPUTATION_FAILED)
    assert lib.gfh_sample_workspace_size(0, 10) == lib.gfh_sample_workspace_size(1, 2 ** 19 + 1) == 0
    assert 0 < lib.gfh_sample_workspace_size(1, 10) < lib.gfh_sample_workspace_size(3, 50257)


def test_packed_struct():
    from ghostflow_hip import _lib as L, ops
    s = L.Sampling.from_buffer_copy(ops._SAMPLING.pack(1, 2, 3, 4, 5.0, 6, 7.0, 8.0))
    assert [getattr(s, f) for f, _ in L.Sampling._fields_] == [1, 2, 3, 4, 5.0, 6, 7.0, 8.0]


def test_python_checks():
    import ghostflow_hip as gh
    with pytest.raises(gh.GhostFlowError):
        gh.sample(torch.zeros(2, 8), torch.zeros(2))
