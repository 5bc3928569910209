"""The C++ surface of the new-token operators and the block-scaled cache, through tests/cpp/test_new_tokens.cpp."""

import pytest

from test_cpp_api import _run


def test_cpp_new_tokens_host():
    _run("cpu", "test_new_tokens")


@pytest.mark.gpu
def test_cpp_new_tokens_device():
    _run("gpu", "test_new_tokens")
