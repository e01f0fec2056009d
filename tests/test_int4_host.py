"""Host side of the 4-bit cache: what its C entry points and wrappers refuse before any launch."""

import ctypes

import pytest
import torch

from mla_kv_quant_b200 import _lib, build, int4


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.load()


def _cache(**kw):
    # addresses that are never followed: every call here returns before a launch
    fields = dict(codes=1 << 20, params=2 << 20, rope=3 << 20, box_center=None, box_radius=None, box_exps=None, num_slots=128, latent_dim=512, rope_dim=64)
    return _lib.Int4Cache(**{**fields, **kw})


@pytest.mark.parametrize("change,code,message", [
    (dict(latent_dim=384), _lib.ROLAQ_EUNSUPPORTED, b"latent_dim"),
    (dict(rope_dim=48), _lib.ROLAQ_EUNSUPPORTED, b"rope_dim"),
    (dict(codes=None), _lib.ROLAQ_EINVAL, b"non-NULL"),
    (dict(params=(2 << 20) + 8), _lib.ROLAQ_EINVAL, b"aligned"),
    (dict(num_slots=100), _lib.ROLAQ_EINVAL, b"num_slots"),
    (dict(num_slots=1 << 31), _lib.ROLAQ_EINVAL, b"num_slots"),
])
def test_a_cache_that_does_not_fit_is_refused(lib, change, code, message):
    c = _cache(**change)
    a = 1 << 24
    for rc in (lib.rolaq_int4_write(a, 0, 512, a, 64, a, 1, 4, ctypes.addressof(c), None, None),
               lib.rolaq_int4_read(ctypes.addressof(c), a, 1, 4, a, 0, 512, None, 0, None, None),
               lib.rolaq_int4_decode(a, 16 * 576, 0, 576, 1, 1, 16, ctypes.addressof(c), a, 1, 1, a, 0.1, a, 1 << 30, a, 16 * 512, 0, 512, None, None, None)):
        assert rc == code and message in lib.rolaq_last_error()


def test_arguments_out_of_range_are_refused(lib):
    c, a = _cache(), 1 << 24
    r = ctypes.addressof(c)
    decode = lambda **k: lib.rolaq_int4_decode(*{**dict(q=a, sb=16 * 576, st=0, sh=576, b=1, t=1, h=16, c=r, pt=a, ps=4, mp=4, sl=a, sm=0.1, ws=a, wb=1 << 30, o=a, ob=16 * 512, ot=0, oh=512, lse=None, err=None, s=None), **k}.values())  # noqa: E731
    for change in (dict(b=-1), dict(b=65536), dict(t=0), dict(t=65), dict(h=0), dict(h=129), dict(mp=-1), dict(sm=-1.0), dict(sm=float("nan")), dict(sm=float("inf")), dict(q=None), dict(sl=None), dict(o=None), dict(ws=None), dict(pt=None), dict(ps=3), dict(sh=568), dict(sh=580), dict(q=a + 2), dict(o=a + 8), dict(oh=504), dict(ob=-8), dict(wb=100)):
        assert decode(**change) == _lib.ROLAQ_EINVAL, change
    assert decode(b=0) == _lib.ROLAQ_OK
    write = lambda **k: lib.rolaq_int4_write(*{**dict(c=a, f=0, ld=512, pe=a, lp=64, sl=a, s64=1, n=4, r=r, err=None, s=None), **k}.values())  # noqa: E731
    for change in (dict(n=-1), dict(n=1 << 31), dict(c=None), dict(pe=None), dict(sl=None), dict(ld=504), dict(ld=516), dict(lp=32), dict(c=a + 8)):
        assert write(**change) == _lib.ROLAQ_EINVAL, change
    assert write(n=0) == _lib.ROLAQ_OK
    assert lib.rolaq_int4_update_boxes(r, a, a, 4, None, None) == _lib.ROLAQ_EINVAL and b"no page boxes" in lib.rolaq_last_error()
    boxed = _cache(box_center=4 << 20, box_radius=5 << 20, box_exps=6 << 20)
    rb = ctypes.addressof(boxed)
    select = lambda **k: lib.rolaq_int4_select_pages(*{**dict(q=a, sb=16 * 576, sh=576, b=1, h=16, c=rb, pt=a, ps=4, mp=4, sl=a, budget=4, kf=1, kl=2, ws=a, wb=1 << 30, t=a, ts=4, n=a, err=None, s=None), **k}.values())  # noqa: E731
    for change in (dict(b=-1), dict(h=0), dict(c=r), dict(budget=2), dict(budget=0), dict(kf=-1), dict(kl=0), dict(kf=2**31 - 1), dict(ps=3), dict(ts=3), dict(wb=100), dict(q=None), dict(t=None), dict(n=None)):
        assert select(**change) == _lib.ROLAQ_EINVAL, change
    assert select(b=0) == _lib.ROLAQ_OK
    assert lib.rolaq_int4_read_boxes(rb, a, 4, a, a, 574, None, None) == _lib.ROLAQ_EINVAL


def test_workspace_sizes(lib):
    sizes = [lib.rolaq_int4_workspace_bytes(b, t, h, 512, p) for b, t, h, p in ((1, 1, 16, 1), (64, 1, 16, 256), (128, 8, 128, 2048))]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for bad in ((-1, 1, 16, 512, 1), (1, 0, 16, 512, 1), (1, 1, 129, 512, 1), (1, 1, 16, 384, 1), (1, 1, 16, 512, -1)):
        assert lib.rolaq_int4_workspace_bytes(*bad) == -1


def test_views_check_their_tensors():
    codes, params, rope = torch.zeros(64, 256, dtype=torch.uint8), torch.zeros(64, 4, 2), torch.zeros(64, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="codes"):
        int4.Int4View(codes.int(), params, rope)
    with pytest.raises(TypeError, match="params"):
        int4.Int4View(codes, params[:, :2], rope)
    with pytest.raises(TypeError, match="rope"):
        int4.Int4View(codes, params, rope.float())
    with pytest.raises(ValueError, match="multiple of 64"):
        int4.Int4View(codes[:63], params[:63], rope[:63])
    with pytest.raises(ValueError, match="contiguous"):
        int4.Int4View(codes, params, torch.zeros(64, 128, dtype=torch.bfloat16)[:, :64])
    with pytest.raises(TypeError, match="boxes"):
        int4.Int4View(codes, params, rope, (torch.zeros(1, 576), torch.zeros(1, 576), torch.zeros(1, 2)))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        int4.Int4View(codes, params, rope)
    with pytest.raises(ValueError, match="pool size"):
        int4.Int4LatentPool(100, 1, device="cpu")
