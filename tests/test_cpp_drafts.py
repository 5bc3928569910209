"""The C++ surface of the drafted-token operators, through tests/cpp/test_drafts.cpp."""

import pytest

from test_cpp_api import _run


def test_cpp_drafts_host():
    _run("cpu", "test_drafts")


@pytest.mark.gpu
def test_cpp_drafts_device():
    _run("gpu", "test_drafts")
