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
