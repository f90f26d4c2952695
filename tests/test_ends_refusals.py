"""CPU tests of what the operators at the ends of a model refuse, beside ``test_ends_host``."""

from test_host import built_lib  # noqa: F401


def test_wait_limit_refuses_a_negative_pair(built_lib):  # noqa: F811
    L = built_lib
    assert L.cb_linear_ce_set_wait_limit(0, -1) == 1 and L.cb_linear_ce_set_wait_limit(1000, 3) == 0
    assert L.cb_linear_ce_set_wait_limit(0, 0) == 0
