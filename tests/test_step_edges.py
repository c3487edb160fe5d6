"""Refusals and sizes of the operators of a serving step over shared pages that the other tests do not reach, without a GPU."""
import itertools
import random

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


def test_chunk_workspaces_of_any_size_fit_what_the_header_says():
    """Steps of any n, rows and max_rows over tables of any width; smaller calls may need more than larger ones, none more than this."""
    rng, most, some = random.Random(5), 40 << 20, 0
    for _ in range(20000):
        d, Hk, G = rng.choice((32, 64, 128)), rng.randint(1, 16), rng.randint(1, 8)
        n, longest = int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 14))
        rows, blocks = rng.randint(1, n * longest) if rng.random() < 0.7 else min(n * longest, n + rng.randint(0, 300)), int(2 ** rng.uniform(0, 12))
        try:
            size = pkg.chunk_attention_workspace(n, rows, longest, Hk * G, pkg.KvCache(AT, Hk * 2 * 64 * d, AT, blocks, 9, Hk, d))
        except pkg._lib.ShahdError as e:
            assert "too many rows or key blocks" in str(e)
            continue
        assert 0 <= size <= most, (d, Hk, G, n, longest, rows, blocks, size)
        some += size > most // 2
    assert some > 20  # the bound is not far above what there is
    grows = [pkg.chunk_attention_workspace(n, rows, longest, 16, pkg.KvCache(AT, 4 * 2 * 64 * 64, AT, 64, 9, 4, 64)) for n, rows, longest in ((16, 32768, 2048), (1, 96, 96))]
    assert grows[0] < grows[1]
