"""Gradients whose tiles one launch cannot hold, without a GPU."""
import pytest

from forward_amd import lib

pytestmark = pytest.mark.skipif(lib.dll.fwdmi_device_count() > 0, reason="made-up addresses: only where nothing can be launched")


@pytest.mark.parametrize("dtype", [lib.F32, lib.F16, lib.BF16])
def test_both_products_are_held_to_the_limit_of_each(dtype):
    """dx and dw together, which one launch may compute, are refused exactly where one of them alone is."""
    d, p, big = lib.dll, 1 << 20, (1 << 64) - 1
    call = lambda m, n, k, dx, dw, db: d.fwdmi_linear_backward(None, m, n, k, p, p, p, None, dx, dw, db, 0, dtype, p, big)
    seen = set()
    for m, n in ((33, 33), (40, 48), (64, 2), (300, 300)):
        for k in (1 << 12, 1 << 26, (1 << 27) - 8, 1 << 28, 1 << 29, (1 << 30) - 1, 1 << 30):
            alone = {call(m, n, k, p, None, None), call(m, n, k, None, p, None)}
            # (ERR_HIP: no device here, it got as far as the launch)
            assert alone <= {lib.ERR_HIP, lib.ERR_UNSUPPORTED}
            want = lib.ERR_UNSUPPORTED if lib.ERR_UNSUPPORTED in alone else lib.ERR_HIP
            assert call(m, n, k, p, p, None) == want, (m, n, k)
            seen.add(want)
    assert len(seen) == 2
