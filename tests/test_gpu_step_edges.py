"""The operators of a serving step over shared pages at the ends of their ranges: values, layouts and buffers that the other tests do not reach."""
import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests.test_gpu_serving_ops import BF16, CODE, F16, F32, _gen, _ints, _normal, _stream  # noqa: E402


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert pkg.load().ShahdDeviceErrorFlag() == 0


# ---- logits --------------------------------------------------------------------------------------------------------

REPETITIONS = [1.3, 0.7, 3.0, 1e-30, 1e-39, 2.0**-149, 1.7e38, 3.4e38]  # below 2^-128 and above 2^126 a reciprocal leaves the range


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("each", [1, 80], ids=["rows on their own", "rows of a sequence together"])
def test_repetition_is_one_division_or_one_product(dtype, each):
    """Where nothing else is asked for, a known token's logit is the 32-bit quotient or product, bit for bit."""
    g, V, n = _gen(41), 4000, len(REPETITIONS)
    x = (_normal(g, n * each, V) * 3).to(dtype)
    x[:, 0], x[:, 2] = 2.0**-24, -(2.0**-24)  # quotients by small numbers stay finite in 32 bits
    history, held, seqs = _ints(list(range(0, V, 2)) * n), _ints([V // 2] * n), _ints(np.arange(n * each) // each)
    rep = torch.tensor(REPETITIONS, dtype=F32)
    out, dev = torch.empty_like(x), rep.cuda()
    pkg.adjust_logits(CODE[dtype], x.data_ptr(), out.data_ptr(), n * each, V, n, sequences=seqs.data_ptr(), history=history.data_ptr(), history_stride=V // 2,
                      history_lengths=held.data_ptr(), repetition=dev.data_ptr(), stream=_stream())
    wide = x.float().cpu()
    r = rep.repeat_interleave(each)[:, None]
    want = torch.where(wide > 0, wide / r, wide * r)
    want[:, 1::2] = wide[:, 1::2]
    assert bool(want[:, ::2].isfinite().any(1).all())
    assert torch.equal(out.cpu(), want.to(dtype))
