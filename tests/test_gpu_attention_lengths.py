"""shahd_attention_set_lengths takes the lengths over before it returns, whatever memory they lie in."""
import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n", [3, 1500])
@pytest.mark.parametrize("pinned", [True, False])
def test_set_lengths_does_not_read_the_array_after_it_returned(pinned, n):
    H, d, C = 2, 32, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), pkg.FusedAttention(n, H, H, d, C, 0.0) as op:
        k, v = (torch.randn(n, 20, H, d, generator=g, device="cuda") for _ in range(2))
        out = torch.empty(n * 20, H, d, device="cuda")
        op.prefill(k.data_ptr(), k.data_ptr(), v.data_ptr(), n, 20, out.data_ptr(), stream.cuda_stream)
        lengths = torch.tensor([5 + i % 7 for i in range(n)], dtype=torch.int32)
        want = lengths.clone()
        if pinned:
            lengths = lengths.pin_memory()
        q = torch.randn(n, H, d, generator=g, device="cuda")
        got = torch.empty_like(q)
        a = torch.zeros(6144, 6144, device="cuda")
        stream.synchronize()
        for _ in range(40):  # some milliseconds, so that the copy would come after the array's next use
            a = a @ a
        op.set_lengths(lengths.numpy(), stream.cuda_stream)
        lengths.fill_(1)
        op.decode(q.data_ptr(), q.data_ptr(), q.data_ptr(), n, got.data_ptr(), stream.cuda_stream)
        stream.synchronize()
        assert [op.length(i) for i in range(n)] == [int(x) + 1 for x in want]
        for i in {0, 1, 2, n // 2, n - 1}:
            L = int(want[i])
            kk, vv = torch.cat([k[i, :L], q[i:i + 1]]).bfloat16().double(), torch.cat([v[i, :L], q[i:i + 1]]).bfloat16().double()
            p = torch.softmax(torch.einsum("hd,lhd->hl", q[i].double(), kk) * d ** -0.5, 1)
            w = torch.einsum("hl,lhd->hd", p, vv)
            # the operator's own bar: 2e-2 of the output's range
            assert float((got[i].double() - w).abs().max()) < 2e-2 * float(w.max() - w.min())


def test_set_lengths_leaves_the_current_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    with pkg.FusedAttention(2, 2, 2, 32, 64, device=1) as op:
        torch.cuda.set_device(0)
        op.set_lengths([3, 4])
        assert torch.cuda.current_device() == 0
        assert (op.length(0), op.length(1)) == (3, 4)
