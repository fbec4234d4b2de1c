"""The Python mirror's paged cache: what it takes for whole pages."""
import pytest


def _rest(streams=2, pages=3):
    import torch
    return torch.zeros(streams, pages, dtype=torch.int32), torch.zeros(streams, dtype=torch.int32), torch.zeros(streams + 1, dtype=torch.int32)


def test_strides_of_axes_of_one(z2):
    """An axis of one element has no stride to speak of: torch gives it any."""
    import torch
    base = torch.zeros(5, 16, 1, 64)
    k = v = base.transpose(1, 2)                       # [5, 1, 16, 64]: one key head, its axis' stride is 64
    assert k.stride() == (1024, 64, 64, 1)
    c = z2.PagedCache(k, v, *_rest())
    assert (c._c.n_pages, c._c.n_kv_heads, c._c.page_size, c._c.head_dim, c._c.page_stride) == (5, 1, 16, 64, 1024)
    k, v = torch.zeros(1, 2, 16, 64), torch.zeros(7, 2, 2, 16, 64)[:1, 1]
    assert k.stride(0) != v.stride(0)                  # one page: nothing lies behind it
    assert z2.PagedCache(k, v, *_rest())._c.page_stride == 2048
    for bad in (torch.zeros(5, 2, 64, 16).transpose(2, 3), torch.zeros(5, 16, 2, 64).transpose(1, 2), torch.zeros(5, 2, 16, 128)[..., :64],
                torch.zeros(5, 2, 32, 64)[:, :, :16]):
        with pytest.raises(ValueError):
            z2.PagedCache(bad, bad, *_rest())
    with pytest.raises(ValueError):
        z2.PagedCache(torch.zeros(5, 2, 16, 64), torch.zeros(5, 4, 16, 64)[:, :2], *_rest())


@pytest.mark.parametrize("scale", [2.5e38, 3.4e38, -1.0, 0.0, float("inf"), float("nan")])
def test_scales_that_leave_f32(z2, scale):
    """The kernels take scores times log2(e): a scale whose product with it is not finite is refused, before CUDA is touched."""
    import ctypes as C
    P = 1 << 20
    c = z2._Cache(P, 2 * P, z2.BF16, 10, 16, 2, 64, 2048, P, 3, 4, P, P)
    assert z2.lib().zonos2cu_cache_attend(C.addressof(c), 5, 8, P, 512, scale, 0, P, 8, 0, 2 * P, 512, None) == z2.EINVAL
