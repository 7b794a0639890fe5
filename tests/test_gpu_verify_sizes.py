"""GPU: verification of drafts at the sizes where a wave takes several parts of a
row, a workgroup several pieces of a sum and a row has more statistics than a wave
has lanes.  Definition, and how far borders are kept away, as in
test_gpu_verify_drafts."""
import numpy as np
import pytest

from test_gpu_verify_drafts import Case
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def parts_to_a_wave(c):
    """As many as bring the first launch down to 2,048 workgroups, at most 8."""
    most = c.n_tok * (1 if c.q is None else 2) * -(-c.vocab // 4096)
    return 1 if most < 2048 else min(most // 2048, 8)


def unlike_parts(c, seed):
    """Rows whose largest logit comes early or late, with whole parts masked and
    some of NaN, and sequences at temperatures of their own."""
    r = np.random.default_rng(seed)
    V = c.vocab
    for x in (c.p,) if c.q is None else (c.p, c.q):
        for t in range(c.n_tok):
            kind = t % 6
            first = int(r.integers(0, max(1, V // 1024 - 3))) * 1024
            if kind == 1:
                x[t, first:first + 1024 * int(r.integers(1, 4))] = -np.inf
            elif kind == 2:
                x[t, :V // 2] = -np.inf
            elif kind == 3:
                x[t, :V] += c.typed(np.linspace(0, 12, V))            # the running maximum moves all along
                x[t] = c.typed(x[t])
            elif kind == 4:
                x[t, first:first + 2048] = np.nan
            elif kind == 5:
                x[t, int(r.integers(V - 900, V))] = 60.0              # all else below 2^-60
    c.t = r.choice(np.array([0, 0.6, 1, 1, 1.7], np.float32), c.n_seq)
    c.u[r.random(c.n_tok) < 0.6] *= np.float32(2.0 ** -12)           # some drafts accepted without q too
    return c


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("drafts,counts,vocab,parts", [
    (True, [3, 5, 0, 4] * 5, 151937, 2),
    (False, [3, 8, 1, 4] * 7, 151937, 2),
    (False, [1] * 400, 50257, 2),
    (True, [5, 1, 6] * 60, 40961, 3),
    (False, [9, 7] * 65, 65535, 8),
])
def test_several_parts_to_a_wave(eng, dtype, drafts, counts, vocab, parts):
    c = Case(counts, vocab, drafts, dtype, seed=vocab % 1000, pad=3 if dtype == "f32" else 7)
    assert parts_to_a_wave(c) >= parts
    unlike_parts(c, len(counts)).check(eng)


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_statistics_than_lanes(eng, dtype, drafts):
    c = Case([3, 2, 1], 270001, drafts, dtype, seed=5)
    assert parts_to_a_wave(c) == 1 and -(-c.vocab // 4096) > 64
    c.p[0, :200000] = -np.inf
    c.p[3, 100:] = -np.inf
    c.check(eng)
    c.t = np.zeros(3, np.float32)
    c.check(eng)


def test_infinite_logits_in_a_later_part(eng):
    c = Case([2] * 60, 151937, False, seed=9)
    assert parts_to_a_wave(c) >= 2
    for t in range(0, c.n_tok, 2):
        c.p[t, 1024 + 17 * t] = c.p[t, 1500 + 1024 * (t % 140)] = np.inf
    c.check(eng)


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_token_each_beside_a_draft_model(eng, temperature):
    """No ranges and nothing drafted: the draft model's rows are of no account."""
    c = Case([1] * 70, 3000, True, temperature=temperature, seed=4)
    c.q[:] = np.nan
    c.check(eng, bare=True)
