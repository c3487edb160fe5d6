"""From the serving operators to FusedAttention's own decode steps over one cache: the rotation has to be the same on both sides,
the operator's own or, with an operator that turns nothing, the caller's."""
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests import serving_refs as R  # noqa: E402
from tests.test_gpu_serving_ops import BF16, F32, _gen, _ints, _no_device_error, _normal, _offsets, _prompt, _rows, _stream  # noqa: E402, F401


@pytest.mark.parametrize("layout,rotary,base,own", [("interleaved", 64, 10000.0, True), ("half", 64, 500000.0, False), ("half", 32, 10000.0, False)])
def test_decode_goes_on_from_appended_prompts(layout, rotary, base, own):
    H, Hk, d, lens = 16, 4, 64, [130, 1, 64]
    n, N, g = len(lens), sum(lens), _gen(81)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), pkg.FusedAttention(n, H, Hk, d, 256, rope_base=base if own else 0.0) as op, pkg.Rope(d, rotary, layout, base=base) as rope:
        st = _stream()
        q, k, v = (_normal(g, N, h, d, dtype=BF16) for h in (H, Hk, Hk))
        off, pos = _ints(_offsets(lens)), _ints([i for t in lens for i in range(t)])
        rope.apply(pkg.BF16, N, pos.data_ptr(), q=_rows(q), q_out=_rows(q), num_heads=H, k=_rows(k), k_out=_rows(k), kv_heads=Hk, v=_rows(v), cache=op.cache(),
                   offsets=off.data_ptr(), n=n, stream=st)
        op.set_lengths(lens, st)
        q1, k1, v1 = (_normal(g, n, h, d) for h in (H, Hk, Hk))
        at, out = _ints(lens), torch.empty_like(q1)
        freq = R.frequencies(rotary, base)
        (qw, _), (kw, _) = R.rotate(q1, at, freq, layout), R.rotate(k1, at, freq, layout)
        if not own:
            rope.apply(pkg.F32, n, at.data_ptr(), q=_rows(q1), q_out=_rows(q1), num_heads=H, k=_rows(k1), k_out=_rows(k1), kv_heads=Hk, stream=st)
        op.decode(q1.data_ptr(), k1.data_ptr(), v1.data_ptr(), n, out.data_ptr(), st)
        side.synchronize()
        for s, t in enumerate(lens):
            rows = slice(sum(lens[:s]), sum(lens[:s]) + t)
            kk, vv = torch.cat([k[rows], kw[s:s + 1].to(BF16)]), torch.cat([v[rows], v1[s:s + 1].to(BF16)])
            want, _ = R.attend(qw[s:s + 1], kk, vv, torch.ones(1, t + 1, dtype=torch.bool, device="cuda"), d ** -0.5, F32)
            # the operator's own bar: 2e-2 of the output's range
            assert float((out[s].double() - want[0]).abs().max()) < 2e-2 * float(want.max() - want.min())
