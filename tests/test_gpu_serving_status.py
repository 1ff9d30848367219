"""What a kernel on pages has left out is told as that by whichever call reads the device's status word next."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


def leave_out(dev, pkg):
    cache = u.Paged(pkg, 3, [(4, 40)], 2, 64, 16, "bf16", "bf16")
    cache.table[0, 2] = cache.pages
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=u.GPU)
    dev.kv_page_append(cache.view(), cache.batch(), pkg.capi.BF16, u.ptr(k), u.ptr(k), stream=u.stream())
    torch.cuda.synchronize()


def test_by_an_operator_on_host_memory(dev, pkg):
    x = np.zeros((4, 64), np.float32)
    y = np.empty_like(x)
    leave_out(dev, pkg)
    with pytest.raises(pkg.hal.KernelError, match="left it out"):
        dev.softmax_host(pkg.capi.F32, 4, 64, x.ctypes.data, y.ctypes.data)
    dev.softmax_host(pkg.capi.F32, 4, 64, x.ctypes.data, y.ctypes.data)
    assert (y == 1 / 64).all() and dev.status() == 0


def test_by_a_stream(dev, pkg):
    leave_out(dev, pkg)
    assert pkg.capi.lib().tsm100_stream_synchronize(dev._h, None) == pkg.capi.ERR_INVALID
    assert "left it out" in pkg.capi.last_error() and dev.status() == 0
