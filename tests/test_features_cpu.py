"""CPU: what the operators on learned inputs and the draws refuse, before anything reaches a GPU: through the C ABI (sizes, strides,
types, settings, workspaces; nothing is launched) and through the Python wrappers (no CPU tensors)."""
import ctypes as C

import pytest

torch = pytest.importorskip('torch')

from bayesian_optimization_amd import _lib as L  # noqa: E402

P = C.c_void_p(4096)      # stands for a device pointer: a refused call never looks at it


@pytest.fixture(scope='module')
def lib():
    return L.load()


def norm(lib, **kw):
    a = dict(device=0, stream=None, dtype=L.TYPE_F32, x=P, xs=8, rows=4, cols=8, w=P, b=P, eps=1e-5, y=P, ys=8, mean=P, rstd=P)
    a.update(kw)
    return lib.gpbo_layernorm(*a.values())


def norm_back(lib, **kw):
    a = dict(device=0, stream=None, dtype=L.TYPE_F32, dy=P, dys=8, x=P, xs=8, rows=4, cols=8, w=P, mean=P, rstd=P, dx=P, dxs=8, dw=P, db=P,
             work=P, nbytes=lib.gpbo_layernorm_backward_workspace(L.TYPE_F32, 4, 8))
    a.update(kw)
    return lib.gpbo_layernorm_backward(*a.values())


def gated(lib, **kw):
    a = dict(device=0, stream=None, dtype=L.TYPE_BF16, act=0, x=P, xs=8, rows=4, cols=8, wg=P, wu=P, ws=8, hidden=16, h=P, hs=16, kg=P, ku=P,
             work=P, nbytes=1 << 30)
    a.update(kw)
    return lib.gpbo_gated(*a.values())


def gated_back(lib, **kw):
    a = dict(device=0, stream=None, dtype=L.TYPE_BF16, act=0, dh=P, dhs=16, x=P, xs=8, rows=4, cols=8, wg=P, wu=P, ws=8, hidden=16, kg=P, ku=P,
             dx=P, dxs=8, dwg=P, dwu=P, dws=8, work=P, nbytes=1 << 30)
    a.update(kw)
    return lib.gpbo_gated_backward(*a.values())


def draw(lib, **kw):
    a = dict(device=0, stream=None, dtype=L.TYPE_F64, s=P, stride=10, rows=2, cols=10, u=P, draws=3, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             params=None, index=P, logp=P, work=P, nbytes=1 << 30)
    a.update(kw)
    return lib.gpbo_draw_static(*a.values())


MOST = 2 ** 31 - 1
BIG = MOST + 1


@pytest.mark.parametrize('call,kw', [
    (norm, k) for k in (dict(dtype=L.TYPE_F64), dict(dtype=9), dict(rows=-1), dict(cols=0), dict(cols=BIG, xs=BIG, ys=BIG), dict(rows=BIG), dict(xs=7),
                        dict(ys=7), dict(eps=-1.0), dict(eps=float('nan')), dict(eps=float('inf')), dict(device=-1), dict(device=64), dict(x=None), dict(y=None))
] + [
    (norm_back, k) for k in (dict(dtype=L.TYPE_F64), dict(rows=-1), dict(cols=0), dict(dys=7), dict(xs=7), dict(dxs=7), dict(dy=None), dict(x=None), dict(mean=None),
                             dict(rstd=None), dict(dx=None), dict(rows=4096, work=None), dict(rows=4096, nbytes=8), dict(rows=4096, nbytes=1 << 30, work=C.c_void_p(4097)), dict(device=64))
] + [
    (gated, k) for k in (dict(dtype=L.TYPE_F64), dict(act=2), dict(rows=-1), dict(cols=0), dict(hidden=0), dict(xs=7), dict(ws=7), dict(hs=15), dict(x=None), dict(wg=None),
                         dict(wu=None), dict(h=None), dict(kg=None), dict(ku=None), dict(rows=MOST, hidden=MOST, hs=MOST), dict(device=-1))
] + [
    (gated, dict(rows=8192, cols=100, xs=100, ws=100, hidden=4096, hs=4096, **k)) for k in (dict(work=None), dict(nbytes=8), dict(work=C.c_void_p(4097)))
] + [
    (gated_back, k) for k in (dict(dtype=L.TYPE_F64), dict(act=-1), dict(dhs=15), dict(xs=7), dict(ws=7), dict(dxs=7), dict(dws=7), dict(dh=None), dict(x=None), dict(wg=None),
                              dict(kg=None), dict(ku=None), dict(dwg=None), dict(dwu=None), dict(rows=65536, work=None), dict(rows=65536, nbytes=8), dict(rows=65536, work=C.c_void_p(4097)), dict(device=64))
] + [
    (draw, k) for k in (dict(dtype=4), dict(dtype=-1), dict(rows=-1), dict(cols=0), dict(cols=(1 << 28) + 1, stride=(1 << 28) + 1), dict(draws=-1), dict(stride=9),
                        dict(temperature=-1.0), dict(temperature=float('nan')), dict(temperature=float('inf')), dict(top_k=-1), dict(top_p=1.1), dict(top_p=-0.1),
                        dict(min_p=1.1), dict(min_p=float('nan')), dict(cols=1 << 20, stride=1 << 20, work=None), dict(cols=1 << 20, stride=1 << 20, nbytes=8), dict(s=None), dict(u=None), dict(index=None), dict(device=-1), dict(device=64))
])
def test_bad_arguments_are_refused(lib, call, kw):
    assert call(lib, **kw) == L.ERR_BAD_ARG


def test_workspace_sizes_of_bad_arguments_are_negative(lib):
    assert lib.gpbo_layernorm_backward_workspace(L.TYPE_F64, 4, 8) == -1
    assert lib.gpbo_layernorm_backward_workspace(L.TYPE_F32, 4, 0) == -1
    assert lib.gpbo_gated_workspace(L.TYPE_F32, -1, 8, 8) == -1
    assert lib.gpbo_gated_backward_workspace(L.TYPE_F32, 4, 8, 0) == -1
    assert lib.gpbo_draw_static_workspace(7, 1, 8, 1) == -1
    assert lib.gpbo_draw_static_workspace(L.TYPE_F64, 1, (1 << 28) + 1, 1) == -1
    assert lib.gpbo_draw_static_workspace(L.TYPE_F16, 65536, (1 << 22) + 1, 1) == -1
    assert lib.gpbo_draw_static_workspace(L.TYPE_F16, 65535, (1 << 22) + 1, 1) > 0


def test_nothing_to_do_launches_nothing(lib):
    """No rows, no draws: done without a GPU."""
    assert norm(lib, rows=0) == L.OK
    assert gated(lib, rows=0) == L.OK
    assert draw(lib, rows=0) == L.OK
    assert draw(lib, draws=0) == L.OK


def test_null_contexts_are_refused(lib):
    i, v = C.c_int64(), C.c_double()
    assert lib.gpbo_draw(None, C.byref(v), 1, 1.0, 0, 1.0, 0.0, C.byref(i), None) == L.ERR_BAD_ARG
    assert lib.gpbo_multi_draw(None, C.byref(v), 1, 1.0, 0, 1.0, 0.0, C.byref(i), None) == L.ERR_BAD_ARG
    assert lib.gpbo_lml_inputs(None, C.byref(v), C.byref(v), 1, 1, C.byref(v), 0.1, 0, C.byref(v), None, C.byref(v)) == L.ERR_BAD_ARG


def test_there_is_no_cpu_path():
    from bayesian_optimization_amd import draws, features
    x, w = torch.ones(3, 4), torch.ones(5, 4)
    for call in (lambda: features.layer_norm(x), lambda: features.gated_unit(x, w, w), lambda: draws.sample(x, torch.ones(3, 1, dtype=torch.float64)),
                 lambda: features.layer_norm_backward(x, x, None, x[:, 0], x[:, 0])):
        with pytest.raises(ValueError, match='CPU'):
            call()
    with pytest.raises(TypeError):
        features.layer_norm([[1.0]])
    with pytest.raises(ValueError):
        features.gated_unit(x, w, w, act='tanh')
    with pytest.raises(ValueError):
        features.FeatureMap(0, 1, 1, device='cpu')
