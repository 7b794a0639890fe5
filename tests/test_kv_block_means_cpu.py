"""Block means that were allocated for a cache of another shape are refused:
their planes have other rows than the calls would read and write."""
import pytest

from vxg_amd import engine


class Planes:
    """An engine that hands out addresses and has no context."""
    ctx = None

    class Buf:
        def __init__(self, nbytes):
            self.ptr, self.nbytes = 0x10000, nbytes

    def alloc(self, nbytes):
        return self.Buf(nbytes)


def calls(cache, means):
    return [lambda: cache.block_means(means, 0, 64),
            lambda: cache.attend_blocks(means, 0x1000, 4, 1, 63, 2, 0, 1, 0x1000)]


@pytest.mark.parametrize("n_kv,hd", [(1, 64), (4, 64), (2, 32), (2, 128), (1, 128), (4, 32)])
def test_means_of_another_shape(n_kv, hd):
    eng = Planes()
    cache = engine.KvQ8Cache.over(eng, 0x1000, 0x1000, 0x1000, 0x1000, 64, 2, 64)
    for call in calls(cache, engine.KvBlockMeans(eng, 2, 32, n_kv, hd)):
        with pytest.raises(engine.BackendError, match="block means") as e:
            call()
        assert e.value.code == engine.VXT_E_SHAPE


def test_means_of_the_cache_and_a_callers_own_go_on():
    """As far as the library, which refuses the missing context."""
    eng = Planes()
    cache = engine.KvQ8Cache.over(eng, 0x1000, 0x1000, 0x1000, 0x1000, 64, 2, 64)
    for means in (engine.KvBlockMeans(eng, 2, 32, 2, 64), engine.KvBlockMeans.over(eng, 0x1000, 0x1000, 2, 32)):
        for call in calls(cache, means):
            with pytest.raises(engine.BackendError) as e:
                call()
            assert e.value.code == engine.VXT_E_ARG
