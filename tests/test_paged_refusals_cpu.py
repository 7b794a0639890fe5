"""CPU: preparation of a batch refuses results, norms and biases that are not
aligned to their elements, where it would use them, and no others."""
import pytest

from test_paged_cpu import ARG, PTR, params, prep

USED = [dict(qo=PTR + 2), dict(p=params(gated_q=1), qs=512, go=PTR + 1)] + [
    dict(p=params(**{name: PTR + off})) for name in ("q_norm", "k_norm", "q_bias", "k_bias", "v_bias") for off in (1, 2)]


@pytest.mark.parametrize("kw", USED)
def test_unaligned_pointers_are_refused(kw):
    rc, msg = prep(**kw)
    assert rc == ARG and b"aligned" in msg, (rc, msg)


@pytest.mark.parametrize("kw", [
    dict(go=PTR + 2),                                                     # not gated
    dict(q=None, qo=PTR + 2), dict(q=None, p=params(gated_q=1), go=PTR + 1),      # K and V alone
    dict(q=None, p=params(q_norm=PTR + 2)), dict(q=None, p=params(q_bias=PTR + 2)),
    dict(qo=PTR + 4, p=params(q_norm=PTR + 4, v_bias=PTR + 12)),
])
def test_what_is_not_used_or_aligned_passes(kw):
    rc, msg = prep(**kw)
    assert rc == ARG and b"context" in msg, (rc, msg)
