"""GPU: verification of drafts at weights about 2^-1000 of the largest, below which
a token has no probability, for its acceptance as for the draw: with q(x) = 0 and
u near 1, or without q and u = 0, a draft is accepted iff p(x) > 0."""
import numpy as np
import pytest

from test_gpu_verify_drafts import Case
from vxg_amd import engine

pytestmark = pytest.mark.gpu

V = 900
TOP, X, OTHER = 17, 600, 850


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def exponent(x, m, t):
    return (float(x) - float(m)) / float(t) / np.log(2.0)


def two_tokens(drafts, temperature, m, x):
    """A token of logit m and a drafted one of x; the draft model's own is
    another one."""
    c = Case([2], V, drafts, temperature=temperature, seed=1)
    c.p[:] = -np.inf
    c.p[:, TOP], c.p[:, X] = m, x
    if drafts:
        c.q[:] = -np.inf
        c.q[:, OTHER] = 1.0
    c.tokens[1] = X
    c.u[:] = np.float32(1 - 2.0 ** -24) if drafts else 0.0
    c.un[:] = np.float32(1 - 2.0 ** -24)
    return c


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("temperature", [1e-3, 0.7, 1.0, 30.0])
@pytest.mark.parametrize("e", [-900, -997, -1003, -1010, -1040, -1073, -1100])
def test_accepted_where_it_has_probability(eng, drafts, temperature, e):
    m = np.float32(8.0)
    x = np.float32(m + e * np.log(2.0) * np.float32(temperature))
    assert abs(exponent(x, m, np.float32(temperature)) - e) < 1
    acc, nxt, lens = two_tokens(drafts, temperature, m, x).run(eng)
    good = e > -1000
    # refused: the largest is what is left; accepted: the next row's largest
    assert acc[0] == good and nxt[0] == TOP


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("steps", [1, 2, 5])
@pytest.mark.parametrize("e", [-990, -1030, -1100])
def test_temperatures_that_logits_barely_resolve(eng, drafts, steps, e):
    """A few steps of f32 below the largest are the whole of the range."""
    m = np.float32(16.0)
    x = np.float32(m - steps * 2.0 ** -20)
    t = np.float32(steps * 2.0 ** -20 / (-e * np.log(2.0)))
    assert abs(exponent(x, m, t) - e) < 1
    acc, nxt, _ = two_tokens(drafts, t, m, x).run(eng)
    assert acc[0] == (e > -1000) and nxt[0] == TOP


@pytest.mark.parametrize("drafts", [True, False])
def test_an_infinite_logit_beside_finite_ones(eng, drafts):
    for x, good in ((np.inf, True), (3e38, False)):
        acc, nxt, _ = two_tokens(drafts, 1.0, np.float32(np.inf), np.float32(x)).run(eng)
        assert acc[0] == good
        if not good:
            assert nxt[0] == TOP
