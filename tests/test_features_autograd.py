"""The operators beside torch's autograd: tensors that require gradients are taken off the tape with a warning, parameters in a feature
map without one."""
import warnings

import numpy as np
import pytest

torch = pytest.importorskip('torch')

from bayesian_optimization_amd._device import off_tape  # noqa: E402


def test_what_warns():
    x = torch.ones(3, requires_grad=True)
    with pytest.warns(UserWarning, match='x requires a gradient'):
        off_tape('x', x)
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        off_tape('x', x.detach())
        with torch.no_grad():
            off_tape('x', x)


@pytest.mark.gpu
def test_operators_warn_and_return_the_same():
    from bayesian_optimization_amd import draws, features
    g = torch.Generator(device='cuda').manual_seed(1)
    x, dy, w = (torch.randn(s, generator=g, device='cuda') for s in ((20, 30), (20, 30), (8, 30)))
    u = torch.rand(20, 3, generator=g, device='cuda', dtype=torch.float64)
    y, mean, rstd = features.layer_norm(x)
    _, kept = features.gated_unit(x, w, w, keep=True)
    dh = dy[:, :8].contiguous()
    leaf = lambda t: t.clone().requires_grad_()
    for plain, tracked in ((lambda: features.layer_norm(x, x[0]), lambda: features.layer_norm(leaf(x), leaf(x[0]))),
                           (lambda: features.layer_norm(x, x[0]), lambda: features.layer_norm(x, leaf(x[0]))),
                           (lambda: features.layer_norm_backward(dy, x, None, mean, rstd), lambda: features.layer_norm_backward(dy, leaf(x), None, mean, rstd)),
                           (lambda: (features.gated_unit(x, w, w),), lambda: (features.gated_unit(x, leaf(w), w),)),
                           (lambda: features.gated_unit_backward(dh, x, w, w, kept), lambda: features.gated_unit_backward(dh, x, w, leaf(w), kept)),
                           (lambda: draws.sample(x, u), lambda: draws.sample(leaf(x), u))):
        with warnings.catch_warnings():
            warnings.simplefilter('error')
            want = plain()
            with torch.no_grad():
                quiet = tracked()
        with pytest.warns(UserWarning, match='requires a gradient'):
            got = tracked()
        assert all(torch.equal(a, b) and torch.equal(a, c) and not b.requires_grad for a, b, c in zip(want, got, quiet))


@pytest.mark.gpu
def test_a_feature_map_of_parameters():
    """Parameters of torch, and an optimiser of torch that steps on the gradients returned."""
    from bayesian_optimization_amd import features, hyperopt
    rng = np.random.default_rng(0)
    raw = rng.standard_normal((30, 41)).cumsum(axis=1) / 5.0
    y = np.sin(raw[:, 3])
    x = torch.from_numpy(raw).float().cuda()
    fmap, other = (features.FeatureMap(41, 16, 3, seed=1) for _ in range(2))
    fmap.params = {k: torch.nn.Parameter(v) for k, v in fmap.params.items()}
    theta = np.array([0.9, 1.1, 1.3])
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        nll, g_theta, grads = hyperopt.lml_features(fmap, x, y, theta, 0.3)
        want, g_want, grads_want = hyperopt.lml_features(other, x, y, theta, 0.3)
        assert nll == want and np.array_equal(g_theta, g_want) and all(torch.equal(grads[k], grads_want[k]) for k in grads)
        assert np.array_equal(fmap.numpy(raw), other.numpy(raw)) and not fmap.forward(x).requires_grad
    step = torch.optim.SGD(fmap.params.values(), lr=1e-4)
    for k, p in fmap.params.items():
        p.grad = grads[k]
    step.step()
    assert hyperopt.lml_features(fmap, x, y, theta, 0.3)[0] < nll
    with pytest.warns(UserWarning, match='x requires a gradient'):
        fmap.forward(x.clone().requires_grad_())
