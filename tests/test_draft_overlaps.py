"""CPU checks of results that may lie where inputs do, and of those that may not."""

import pytest

from test_draft_checks import P, _refused, vla  # noqa: F401 (the fixture)


@pytest.mark.parametrize("kw", [dict(qo=P, q=P, ldq=256, ldqo=512), dict(qo=P, q=P, ldq=512, ldqo=256), dict(ko=P, k=P, ldk=128, ldko=256),
                                dict(ko=P, k=P, ldk=640, ldko=128, cache=None)])
def test_append_in_place_keeps_its_strides(vla, kw):  # noqa: F811
    """Rows written at another stride would lie over rows that other blocks still read."""
    args = dict(qo=2 * P, q=P, ko=None, k=3 * P, v=4 * P)
    args.update(kw)
    assert "same stride" in _refused(vla, "vla_rope_kv4_append_dev", args)
