"""GPU: verification of drafts whose token ranges fall, or lie partly outside of
the batch: no sequence has tokens in the first case, whatever an earlier call left
in the workspace; in the second they are cut to the batch's."""
import numpy as np
import pytest

from test_gpu_verify_drafts import NONE, Case
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def fill_workspace(eng, c, drafts):
    """Statistics of other rows, with ids and sums of a larger vocabulary."""
    for t in (0.0, 1.0):
        o = Case([c.n_tok], 4 * c.vocab, drafts, temperature=t, seed=99, tail=2)
        o.p[:, -1] = 99.0
        o.run(eng)


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("start", [[0, 7, 2, 9], [5, 0, 3, 9], [0, 3, 9, 6], [9, 9, 9, 0], [0, 2 ** 31 - 1, 4, 9], [4, 6, -7, 9]],
                         ids=str)
def test_ranges_that_fall_hold_nothing(eng, drafts, temperature, start):
    c = Case([3, 3, 3], 500, drafts, temperature=temperature, seed=3)
    c.start = np.array(start, np.int32)
    for _ in range(2):
        fill_workspace(eng, c, drafts)
        acc, nxt, lens = c.run(eng)
        assert np.all(acc == 0) and np.all(nxt == NONE) and np.array_equal(lens, c.lens)


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("at", [0, 63, 64, 700, 998])
def test_one_fall_among_many_sequences(eng, drafts, at):
    c = Case([2] * 1000, 40, drafts, seed=at, tail=3)
    want = c.run(eng)
    c.start[at + 1] = c.start[at + 2] + 1
    acc, nxt, lens = c.run(eng, in_place=True)
    assert np.all(acc == 0) and np.all(nxt == NONE) and np.array_equal(lens, c.lens)
    c.start[at + 1] = 2 * (at + 1)
    for a, b in zip(want, c.run(eng)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("start,same", [([0, 4, 99, 50], [0, 4, 9, 9]), ([-5, -9, 3, 9], [0, 0, 3, 9]),
                                        ([0, 0, 9, 2 ** 31 - 1], [0, 0, 9, 9])], ids=str)
def test_ranges_are_cut_to_the_batch(eng, drafts, start, same):
    """What falls outside of the batch alone is no fall."""
    c = Case([3, 3, 3], 500, drafts, seed=5)
    c.start = np.array(same, np.int32)
    c.counts = np.diff(c.start)
    want = c.want()
    c.start = np.array(start, np.int32)
    for w, g in zip(want, c.run(eng)):
        assert np.array_equal(w, g)
