"""Numbers of the serving operators' calls that are fine in 64 bits but leave the range of the 32 that the kernels take them in are
refused, without a device."""
import pytest

from tests.helpers import pkg

ROWS = pkg.Rows(1 << 20, 128, 64)  # never followed: the calls are refused before
CACHE = pkg.KvCache(1 << 20, 2 * 2 * 64 * 64, 1 << 20, 4, 9, 2, 64)


def _refused(text, call, *args, **kwargs):
    with pytest.raises(pkg._lib.ShahdError, match=text) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg._lib.SHAHD_EINVAL


@pytest.mark.parametrize("scale", [1e-60, 1e-46, 2.4e38, 1e39, 1e300])
def test_scales_beyond_32_bits(scale):
    """0 times the -inf of a masked key would be NaN; so would a score of 0 times an infinite scale."""
    ok = dict(dtype=pkg.BF16, q=ROWS, k=ROWS, v=ROWS, out=ROWS, offsets=1 << 20, n=1, rows=4, num_heads=2)
    _refused("scale must be", pkg.prompt_attention, **ok, kv_heads=2, head_dim=64, scale=scale)
    _refused("scale must be", pkg.tree_attention, **ok, cache=CACHE, lengths=1 << 20, masks=1 << 20, max_nodes=4, scale=scale)


@pytest.mark.parametrize("magnitude", [1e-60, -1e-60, 1e39, -1e39])
def test_rope_magnitudes_beyond_32_bits(magnitude):
    _refused("magnitude", pkg.Rope, 64, magnitude=magnitude)


def test_rope_stretched_bases_beyond_64_bits():
    _refused("stretched", pkg.Rope, 64, base=1e200, scaling="stretched", factor=1e150)
    pkg.Rope(64, base=1e100, scaling="stretched", factor=1e100).close()
