"""Numbers at the ends of their range, refused before any CUDA call."""

import pytest

FAKE = 1 << 20


def attend(m5, **change):
    """The C entry point's code and message for a small batch with `change`d fields."""
    lib, paged, _lib = m5
    f = dict(tokens=3, batch=2, q_heads=4, kv_heads=2, dim=64, starts=FAKE, lens=FAKE, k=FAKE, v=FAKE,
             dtype=_lib.BF16, pages=5, page=16, kp=1024, kh=512, ks=64, vp=1024, vh=512, vs=64,
             table=FAKE, width=1, stride=1, q=FAKE, qt=256, qh=64, out=FAKE, ot=256, oh=64, lse=0,
             longest=2, scale=1.0, softcap=0.0, slopes=0, window=0, prefix=0, ws=0, ws_bytes=0)
    assert set(change) <= set(f)
    f.update(change)
    return lib.m5b_paged_attention(paged._PACK_ATTEND.pack(*f.values()), None), lib.m5b_last_error()


@pytest.fixture
def m5():
    from m5kernels_b200 import _lib, paged

    return _lib.lib(), paged, _lib


@pytest.mark.parametrize("scale", [1e-50, 3e38, 1e300, float("inf"), float("nan"), -1e-50])
def test_scales_that_fp32_does_not_hold(m5, scale):
    code, text = attend(m5, scale=scale)
    assert code == m5[2].EINVAL and b"scale" in text


@pytest.mark.parametrize("change", [dict(tokens=(2**31 - 1) // 4), dict(tokens=2**31 - 1, q_heads=1, kv_heads=1),
                                    dict(q_heads=65535, kv_heads=65535, dim=65535, tokens=1)])
def test_rows_and_channels_beyond_the_index_range(m5, change):
    """What the kernels count in 32 bits, rounded up to tiles of rows."""
    code, text = attend(m5, **change)
    assert code == m5[2].EUNSUPPORTED and b"range" in text
