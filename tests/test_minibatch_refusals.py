"""Calls that the minibatch operators refuse: argument checks come before the device is touched, so they run without a GPU."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import recommender_amd as ra
from recommender_amd import _abi

F = torch.float32


def _x(n=4, d=8, dtype=F):
    return torch.zeros(n, d, dtype=dtype)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("call, error", [
    (lambda: ra.embedding(_x().double(), _i(0)), TypeError),
    (lambda: ra.embedding(_x().half(), _i(0)), TypeError),
    (lambda: ra.embedding(_x(), torch.tensor([0])), TypeError),                 # int64 ids
    (lambda: ra.embedding(torch.zeros(4), _i(0)), ValueError),
    (lambda: ra.embedding(torch.zeros(4, 0), _i(0)), ValueError),
    (lambda: ra.embedding_grad(_x(), _i(0, 1), 4), ValueError),                 # a grad row per id
    (lambda: ra.embedding_grad(_x(2), _i(0, 1), -1), ValueError),
    (lambda: ra.embedding_grad(_x(2), _i(0, 1), 4, accumulate=True), ValueError),
    (lambda: ra.embedding_grad(_x(2), _i(0, 1), 4, out=_x(3)), ValueError),
    (lambda: ra.embedding_grad(_x(2), _i(0, 1), 4, out=_x(4, 8, torch.bfloat16)), ValueError),
    (lambda: ra.embedding_grad(_x(2), _i(0, 1), 4, out=torch.zeros(8, 4).t()), ValueError),
    (lambda: ra.embedding_grad(_x(2), _i(0, 1), 4, out=torch.zeros(8).expand(4, 8)), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5, 7), _i(0, 0, 0, 0)), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5, 8, torch.bfloat16), _i(0, 0, 0, 0)), ValueError),
    (lambda: ra.softmax_loss(_x(4, 257), _x(5, 257), _i(0, 0, 0, 0)), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(0), _i(0, 0, 0, 0)), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0)), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0, 0), scale=0.0), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0, 0), scale=float("inf")), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0, 0), scale=1e-21), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0, 0), bias=torch.zeros(4)), ValueError),
    (lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0, 0), bias=torch.zeros(5).bfloat16()), ValueError),
    (lambda: ra.softmax_loss_grads(_x(), _x(5), _i(0, 0, 0, 0), weights=torch.zeros(3)), ValueError),
    (lambda: ra.grad_norm([]), ValueError),
    (lambda: ra.grad_norm([_x().double()]), TypeError),
    (lambda: ra.grad_norm([torch.zeros(8).expand(4, 8)]), ValueError),
    (lambda: ra.grad_norm([_x(4, 8)[:, :4]]), ValueError),                      # gaps
    (lambda: ra.clip_grads([_x()], 0.0), ValueError),
    (lambda: ra.clip_grads([_x()], float("nan")), ValueError),
    (lambda: ra.clip_grads([_x()], 1.0, out=[_x(5)]), ValueError),
    (lambda: ra.clip_grads([_x()], 1.0, out=[_x(), _x()]), ValueError),
])
def test_python_refusals(call, error):
    with pytest.raises(error):
        call()


def test_out_must_not_overlap():
    both = torch.zeros(8, 8)
    with pytest.raises(ValueError, match="overlap"):
        ra.embedding_grad(both[:4], _i(0, 1, 2, 3), 4, out=both[2:6])


@pytest.mark.parametrize("change, error", [
    (dict(users=np.zeros(4, np.int32)), TypeError), (dict(items=[0, 1, 2, 3]), TypeError),
    (dict(users=torch.zeros(4, dtype=torch.int64)), TypeError), (dict(items=torch.zeros(4)), TypeError),
    (dict(user_vecs=np.zeros((9, 8), np.float32)), TypeError), (dict(item_vecs=np.zeros((5, 8))), TypeError),
    (dict(user_vecs=_x(9).double()), TypeError), (dict(b_i=np.zeros(5)), TypeError), (dict(b_i=torch.zeros(5).bfloat16()), TypeError),
    (dict(items=_i(0)), ValueError),                                            # one item for all users: not broadcast
    (dict(users=_i(0)), ValueError), (dict(users=_i(0, 1, 2, 3).view(2, 2), items=_i(0, 1, 2, 3).view(2, 2)), ValueError),
    (dict(user_vecs=_x(9, 7)), ValueError), (dict(user_vecs=_x(9, 8, torch.bfloat16)), ValueError), (dict(item_vecs=torch.zeros(8)), ValueError),
    (dict(b_i=torch.zeros(9)), ValueError), (dict(b_i=torch.zeros(1)), ValueError)])
def test_ranking_step_refusals(change, error):
    given = dict(users=_i(0, 1, 2, 3), items=_i(0, 1, 2, 3), user_vecs=_x(9), item_vecs=_x(5), b_i=torch.zeros(5))
    with pytest.raises(error, match="ranking_step"):
        ra.ExplicitMF.ranking_step(**{**given, **change})


def test_ranking_step_tables_of_their_own():
    """One table inside the other, a table that holds an element twice: refused before anything is updated."""
    both, users, items = torch.zeros(12, 8), _i(0, 1), _i(2, 3)
    for user_vecs, item_vecs, b_i in ((both[:6], both[5:], None), (both, both[:11], None), (torch.zeros(1, 8).expand(9, 8), both, None),
                                      (_x(9), torch.zeros(1, 8).expand(5, 8), None), (_x(9), both, torch.zeros(1).expand(12)),
                                      (_x(9), both, both.view(-1)[:12]), (_x(9), both, both[:, 7]), (both[:, :5], both[:, 3:], None),
                                      (both[:, 1:5], both[:, :4], None), (_x(9), torch.zeros(20).as_strided((5, 8), (3, 1)), None)):
        with pytest.raises(ValueError, match="share memory|element twice"):
            ra.ExplicitMF.ranking_step(users, items, user_vecs, item_vecs, b_i)


def test_ranking_step_columns_of_one_table_are_apart():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    wide, users, items = torch.zeros(12, 17), _i(0, 1), _i(2, 3)
    for user_vecs, item_vecs, b_i in ((wide[:, :8], wide[:, 8:16], wide[:, 16]), (wide[:5, 9:], wide[:, 1:9], wide[:, 0]), (wide, wide, None)):
        with pytest.raises(_abi.MfsgdError, match="no ROCm GPU"):               # nothing else is wrong with the call
            ra.ExplicitMF.ranking_step(users, items, user_vecs, item_vecs, b_i)


def test_no_gpu_no_answer():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    for call in (lambda: ra.embedding(_x(), _i(0)), lambda: ra.embedding_grad(_x(1), _i(0), 4),
                 lambda: ra.softmax_loss(_x(), _x(5), _i(0, 0, 0, 0)), lambda: ra.clip_grads([_x()], 1.0)):
        with pytest.raises(_abi.MfsgdError):
            call()


def _refused(rc):
    assert rc == -1, rc                    # MFSGD_ERR_ARG
    return _abi.lib().mfsgd_last_error().decode()


def test_c_refusals_embedding():
    lib, p = _abi.lib(), 0x1000
    assert "shape" in _refused(lib.mfsgd_hip_embedding(p, 7, 4, 8, p, 1, 1.0, 0, p, None))          # stride < d
    assert "shape" in _refused(lib.mfsgd_hip_embedding(p, 8, 4, 0, p, 1, 1.0, 0, p, None))
    assert "dtype" in _refused(lib.mfsgd_hip_embedding(p, 8, 4, 8, p, 1, 1.0, 2, p, None))
    assert "null" in _refused(lib.mfsgd_hip_embedding(p, 8, 4, 8, None, 1, 1.0, 0, p, None))
    assert lib.mfsgd_hip_embedding(None, 8, 0, 8, None, 0, 1.0, 0, None, None) == 0                 # nothing to do
    need = lib.mfsgd_embedding_grad_workspace(5000, 100, 8)
    assert need > 0
    assert lib.mfsgd_embedding_grad_workspace(-1, 100, 8) == -1
    assert lib.mfsgd_embedding_grad_workspace((1 << 31) - 1, 100, 8) == -1
    assert lib.mfsgd_embedding_grad_workspace((1 << 31) - 1023, 100, 8) == -1 and lib.mfsgd_embedding_grad_workspace((1 << 31) - 1024, 100, 8) > 0
    assert lib.mfsgd_embedding_grad_workspace(5000, 100, (1 << 30) + 1) == -1
    assert "shape" in _refused(lib.mfsgd_hip_embedding_grad(p, 8, p, (1 << 31) - 1023, 100, 8, 1.0, 0, 0, p, 8, p, 1 << 50, None))
    assert "workspace" in _refused(lib.mfsgd_hip_embedding_grad(p, 8, p, 5000, 100, 8, 1.0, 0, 0, p, 8, p, need - 1, None))
    assert "workspace" in _refused(lib.mfsgd_hip_embedding_grad(p, 8, p, 5000, 100, 8, 1.0, 0, 0, p, 8, p + 4, need, None))
    assert "workspace" in _refused(lib.mfsgd_hip_embedding_grad(p, 8, p, 5000, 100, 8, 1.0, 0, 0, p, 8, None, need, None))
    assert "shape" in _refused(lib.mfsgd_hip_embedding_grad(p, 8, p, 5000, 100, 8, 1.0, 0, 0, p, 7, p, need, None))
    assert "null" in _refused(lib.mfsgd_hip_embedding_grad(None, 8, p, 5000, 100, 8, 1.0, 0, 0, p, 8, p, need, None))


def test_c_refusals_softmax_loss():
    lib, p = _abi.lib(), 0x1000
    need = lib.mfsgd_softmax_loss_workspace(4, 5, 8, 0, 1)
    assert need > 0
    for bad in ((4, 0, 8, 0), (4, 5, 0, 0), (4, 5, 257, 0), (4, 5, 8, 3), (-1, 5, 8, 0), (1 << 30, 5, 8, 0)):
        assert lib.mfsgd_softmax_loss_workspace(*bad, 1) == -1, bad

    def call(xs=8, ts=8, n=4, items=5, d=8, scale=1.0, dtype=0, dx=p, dw=p, ws=p, nbytes=need):
        return lib.mfsgd_hip_softmax_loss_grads(p, xs, p, ts, p, None, None, 1.0, n, items, d, scale, dtype, p, p, dx, dw, None, ws,
                                                nbytes, None)
    for kw, word in ((dict(xs=7), "shape"), (dict(ts=7), "shape"), (dict(items=0), "shape"), (dict(d=257, xs=257, ts=257), "shape"),
                     (dict(n=1 << 30), "shape"), (dict(dtype=5), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                     (dict(scale=float("nan")), "scale"), (dict(scale=1e-30), "scale"), (dict(ws=None), "workspace"), (dict(ws=p + 8), "workspace"),
                     (dict(nbytes=need - 1), "workspace"), (dict(dx=None), "null"), (dict(dw=None), "null")):
        assert word in _refused(call(**kw)), kw
    assert "null" in _refused(call(n=0, dx=None, dw=None))        # an empty batch still has a table's gradient to write
    assert "null" in _refused(lib.mfsgd_hip_softmax_loss(None, 8, p, 8, p, None, 4, 5, 8, 1.0, 0, p, p, p, need, None))


def test_c_workspace_of_a_table_as_it_is():
    """A bf16 table that is an operand as it is has no copy in the workspace; one that is not needs it, and the call says so."""
    lib, p = _abi.lib(), 0x1000
    size = lambda n, items, d, dtype, flags: lib.mfsgd_softmax_loss_workspace(n, items, d, dtype, flags)    # noqa: E731
    for d, least in ((256, 624961 * 256 * 2), (32, 624961 * 32 * 2)):
        for grads in (0, 1):
            assert size(4096, 624961, d, 1, grads) - size(4096, 624961, d, 1, grads + 2) >= least
    for n, items, d, dtype in ((4096, 9000, 100, 1), (4096, 9000, 64, 0), (3, 9000, 64, 1)):      # padded, split, or converted on the way
        assert size(n, items, d, dtype, 1) == size(n, items, d, dtype, 3)
    need = size(4096, 9000, 64, 1, 3)

    def call(table=p, stride=64, nbytes=need):
        return lib.mfsgd_hip_softmax_loss_grads(p, 64, table, stride, p, None, None, 1.0, 4096, 9000, 64, 1.0, 1, p, p, p, p, None, p, nbytes,
                                                None)
    assert "workspace" in _refused(call(nbytes=need - 1))
    for kw in (dict(table=p + 2), dict(stride=65), dict(stride=1 << 20)):
        assert "workspace" in _refused(call(**kw)), kw


def test_c_refusals_clip():
    lib, p = _abi.lib(), 0x1000
    norm, ws = p + 0x100000, p + 0x200000

    def call(ptrs, sizes, dtypes, outs=None, top=1.0, nbytes=1 << 20, norm=norm, ws=ws):
        n = len(sizes)
        return lib.mfsgd_hip_clip_grads((C.c_void_p * n)(*ptrs), None if outs is None else (C.c_void_p * n)(*outs),
                                        (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*dtypes), n, top, norm, ws, nbytes, None)
    for kw, word in ((dict(ptrs=[p], sizes=[4], dtypes=[0], top=0.0), "max_norm"),
                     (dict(ptrs=[p], sizes=[4], dtypes=[0], top=float("nan")), "max_norm"),
                     (dict(ptrs=[p], sizes=[-1], dtypes=[0]), "negative"),
                     (dict(ptrs=[None], sizes=[4], dtypes=[0]), "null"),
                     (dict(ptrs=[p], sizes=[4], dtypes=[2]), "dtype"),
                     (dict(ptrs=[p], sizes=[4], dtypes=[0], norm=None), "null"),
                     (dict(ptrs=[p], sizes=[4], dtypes=[0], nbytes=8), "workspace"),
                     (dict(ptrs=[p], sizes=[4], dtypes=[0], ws=None), "workspace"),
                     (dict(ptrs=[p, p], sizes=[4, 4], dtypes=[0, 0]), "shares"),                         # the same tensor twice
                     (dict(ptrs=[p, p + 8], sizes=[4, 4], dtypes=[0, 0]), "shares"),
                     (dict(ptrs=[p], sizes=[4], dtypes=[0], outs=[p + 4]), "shares"),                    # shifted onto itself
                     (dict(ptrs=[p, p + 64], sizes=[4, 4], dtypes=[0, 1], outs=[p + 64, p]), "shares"),  # exchanged
                     (dict(ptrs=[p, p + 64], sizes=[4, 4], dtypes=[0, 0], outs=[p + 128, p + 128]), "shares")):
        assert word in _refused(call(**kw)), kw
    sizes = (C.c_int64 * 2)(5, -5)
    assert lib.mfsgd_grad_norm_workspace(sizes, 2) == -1 and lib.mfsgd_grad_norm_workspace(None, 2) == -1
    assert lib.mfsgd_grad_norm_workspace(sizes, 1) > 0


def test_the_package_imports_without_torch():
    code = ("import sys, recommender_amd as ra; assert 'torch' not in sys.modules; ra.embedding; "
            "assert 'torch' in sys.modules and ra.minibatch.clip_grads is ra.clip_grads and not hasattr(ra, 'nothing')")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
