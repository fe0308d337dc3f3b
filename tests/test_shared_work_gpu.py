"""Two threads on streams of their own and an error raised inside a backward pass, run here also in front of the
captured steps of test_wide_gpu.py (files run in the order of their names): what such calls leave behind may not
reach into a later capture."""
import pytest

from test_work_shared_gpu import (  # noqa: F401
    test_dropout_layer_refuses_recomputation, test_operators_from_two_threads)

pytestmark = pytest.mark.gpu
