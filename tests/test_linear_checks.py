"""Forward operators: checks that need no GPU."""
import zkml_b200 as Z


def test_wait_self_test_refuses_null_arguments():
    assert Z.lib().zkml_selftest_linear_wait(None, None, 1, 20) == 1


def test_checked_call_refuses_null_arguments():
    assert Z.lib().zkml_linear_forward_checked(None, None) == 1
