"""Prompt and shared-prefix attention and the page operations at their edges: values that are not numbers, tables that end
before their streams do, batches of many sequences, long prompts, and calls that follow one another without a pause."""
import numpy as np
import pytest
import torch

from helpers import bf16, dev_bf16, host, to_dev
from oracle import paged
from test_paged_attention_gpu import D, PAGE, SCALE, close, make_cache, run_prefill, run_shared, scattered

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


# ---- tables that end before their streams do ----
def test_missing_pages_are_reported(fb):
    """A page below a row's length whose table entry is negative is a sequence longer than its table; entries that no row
    looks at are not."""
    from flint_b200 import prefill_attention as pa
    from flint_b200 import shared_prefix_attention as sp
    fb._lib.check_device_status()
    report = lambda: pytest.raises(fb._lib.FlintError, match="longer than its block table")
    for column, window, bad in ((0, 0, True), (18, 0, True), (12, 70, False), (12, 80, True)):
        args, _ = run_prefill(np.random.default_rng(41), [5, 20], [290, 300], 2, 4, window, False)
        fb._lib.check_device_status()
        args[2][1, column] = -1
        pa.flint_prefill_attention(*args)
        if bad:
            with report():
                fb._lib.check_device_status()
        fb._lib.check_device_status()
    for column, streams, window, bad in ((3, [0, 1, 2], 0, True), (17, [1], 0, True), (3, [0, 1, 2], 64, False),
                                         (17, [0], 0, False)):
        args, _ = run_shared(np.random.default_rng(42), [3], [256], [270, 290, 260], 2, 4, window, False)
        fb._lib.check_device_status()
        args[2][streams, column] = -1
        sp.flint_shared_prefix_attention(*args)
        if bad:
            with report():
                fb._lib.check_device_status()
        fb._lib.check_device_status()
