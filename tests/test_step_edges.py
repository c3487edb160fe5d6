"""Refusals and sizes of the operators of a serving step over shared pages that the other tests do not reach, without a GPU."""
import itertools

import pytest

from tests.helpers import pkg
from tests.test_step_ops import AT, _no_device, _refused


@pytest.mark.parametrize("dtype,size", [(pkg.F32, 4), (pkg.BF16, 2)])
def test_logits_and_results_that_share_memory_in_part(dtype, size):
    ok = dict(dtype=dtype, logits=AT, out=AT, rows=4, vocab=100, n=4)
    call = pkg.adjust_logits
    for shift in (1, 50, 99, 100, 399, -1, -100, -399):
        _refused("overlap", call, **{**ok, "out": AT + shift * size})
    for shift in (400, -400, 4000):
        _no_device(call, **{**ok, "out": AT + shift * size})
    # two halves of one buffer, results in front of or behind their logits: no row meets another
    halves = {**ok, "logits_stride": 200, "out_stride": 200}
    for shift in (100, -100, 300, -300, 700, 701, 799):
        _no_device(call, **{**halves, "out": AT + shift * size})
    for shift in (99, 101, -99, -101, 200, -200, 600, 699, -699):
        _refused("overlap", call, **{**halves, "out": AT + shift * size})


def test_logits_and_results_of_other_strides_that_share_memory():
    """Every pair of small layouts, against a list of what each row holds."""
    rows, vocab = 3, 3
    for a, b, shift in itertools.product(range(3, 9), range(3, 9), range(-26, 27)):
        if shift == 0:
            continue
        held = {i * a + v for i in range(rows) for v in range(vocab)}
        share = any(shift + i * b + v in held for i in range(rows) for v in range(vocab))
        args = dict(dtype=pkg.F32, logits=AT, out=AT + 4 * shift, rows=rows, vocab=vocab, n=rows, logits_stride=a, out_stride=b)
        if share:
            _refused("overlap", pkg.adjust_logits, **args)
        else:
            _no_device(pkg.adjust_logits, **args)
