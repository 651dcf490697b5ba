"""The settings of a draw: each is checked on its own, also beside one that comes as a tensor; none that lies on the GPU is waited for."""
import math

import pytest

torch = pytest.importorskip('torch')

from bayesian_optimization_amd import draws  # noqa: E402

GOOD = dict(temperature=0.5, top_k=3, top_p=0.9, min_p=0.01)
BAD = [('temperature', v) for v in (-1.0, math.nan, math.inf)] + [('top_k', v) for v in (-3, 2.5, math.inf, math.nan)] + [
    (n, v) for n in ('top_p', 'min_p') for v in (1.5, -0.1, math.nan)]


class OnGpu(torch.Tensor):
    """Stands for a tensor on a GPU: whoever looks at its value fails."""
    is_cuda = True

    def item(self):
        raise AssertionError('waited for')
    __float__ = item


@pytest.mark.parametrize('name,value', BAD)
def test_a_number_out_of_range_is_refused_beside_a_tensor(name, value):
    for other in GOOD:
        st = dict(GOOD, **{name: value})
        if other != name:
            st[other] = torch.zeros(2).as_subclass(OnGpu)
        with pytest.raises(ValueError, match=name):
            draws._numbers(tuple(st.values()))
        with pytest.raises(ValueError, match=name):
            draws._numbers(tuple(dict(st, **{name: torch.tensor(value, dtype=torch.float64)}).values()))


def test_numbers_of_tensors():
    assert draws._numbers(tuple(GOOD.values())) == tuple(GOOD.values())
    assert draws._numbers((torch.tensor(2.0), torch.tensor(7), 0.5, torch.tensor(0.25))) == (2.0, 7, 0.5, 0.25)
    assert draws._numbers(tuple(torch.tensor(-9.0).as_subclass(OnGpu) for _ in range(4))) == (1.0, 0, 1.0, 0.0)


@pytest.mark.gpu
def test_settings_on_the_gpu():
    g = torch.Generator(device='cuda').manual_seed(1)
    s, u = torch.randn(4, 3000, generator=g, device='cuda'), torch.rand(4, 30, generator=g, device='cuda', dtype=torch.float64)
    on = lambda v: torch.tensor(v, device='cuda', dtype=torch.float64)
    want = draws.sample(s, u, **GOOD)
    for name in GOOD:
        got = draws.sample(s, u, **dict(GOOD, **{name: on(GOOD[name])}))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
    everything = {k: on(v) for k, v in GOOD.items()}
    draws.sample(s, u, **everything)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):      # would end in an error if one of them were read
        out = draws.sample(s, u, **everything)
    for k in (3, 40, 1, 500):
        everything['top_k'].fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, draws.sample(s, u, **dict(GOOD, top_k=k))))
    for name, value in BAD:
        for other in GOOD:
            if other != name:
                with pytest.raises(ValueError, match=name):
                    draws.sample(s, u, **{other: on(GOOD[other]), name: value})
    with pytest.raises(ValueError):
        draws.sample(s, u, top_k=torch.ones(3, device='cuda'))
    with pytest.raises(ValueError):
        draws.sample(s, u, top_k=torch.ones(4))
