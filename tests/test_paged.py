"""The paged-cache entry points without a GPU: the description's layout, and everything they refuse before a launch."""
import ctypes as C

import pytest
import torch

from amd_c_b200 import _lib
from amd_c_b200 import kernels as K

ARG, SIZE = -1, -2


class Pages(C.Structure):  # as include/ie_b200.h declares it
    _fields_ = [("kp", C.c_void_p), ("vp", C.c_void_p), ("table", C.c_void_p), ("n_pages", C.c_uint32), ("page", C.c_uint32), ("n_kv", C.c_uint32),
                ("hd", C.c_uint32), ("n_seq", C.c_uint32), ("table_cols", C.c_uint32), ("table_stride", C.c_uint32), ("kv_f32", C.c_int),
                ("page_stride", C.c_size_t)]


AT = 1 << 20  # an address that nothing is read from


def pages(**change):
    p = dict(kp=AT, vp=AT, table=AT, n_pages=10, page=16, n_kv=8, hd=128, n_seq=4, table_cols=5, table_stride=5, kv_f32=0, page_stride=16 * 8 * 128 * 2)
    p.update(change)
    return C.cast(C.pointer(Pages(**p)), C.c_void_p)


def rope(lib, p, q=AT, k=AT, v=AT, q_out=AT, cos=AT, sin=AT, n_rope=80, pos=AT, seq=None, nq=32, T=1, stride=48 * 512, out_stride=32 * 512):
    return lib.ie_b200_rope_kv_paged(q, k, v, q_out, p, cos, sin, n_rope, pos, seq, nq, 0, T, stride, out_stride, None, None)


def attn(lib, p, q=AT, out=AT, oq=None, lens=AT, seq=None, n_head=32, R=1, q_stride=4096 * 4, out_stride=4096 * 4, oq_stride=5120, scratch=AT):
    return lib.ie_b200_attn_decode_paged(q, p, out, oq, lens, seq, n_head, R, q_stride, out_stride, oq_stride, scratch, None, None)


def test_the_packed_description_is_the_header_s():
    raw = _lib.KV_PAGES.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 1, 12)
    assert len(raw) == C.sizeof(Pages)
    p = Pages.from_buffer_copy(raw)
    assert [getattr(p, n) for n, _ in Pages._fields_] == [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 1, 12]


BAD_PAGES = [(dict(kp=None), ARG), (dict(vp=None), ARG), (dict(table=None), ARG), (dict(kp=AT + 8), ARG), (dict(vp=AT + 2), ARG), (dict(table=AT + 2), ARG),
             (dict(page_stride=16 * 8 * 128 * 2 + 8), ARG), (dict(kv_f32=2), ARG), (dict(n_pages=0), SIZE), (dict(page=0), SIZE), (dict(n_kv=0), SIZE),
             (dict(hd=0), SIZE), (dict(hd=100), SIZE), (dict(hd=1024), SIZE), (dict(n_seq=0), SIZE), (dict(table_cols=0), SIZE), (dict(table_stride=4), SIZE),
             (dict(page_stride=16 * 8 * 128 * 2 - 16), SIZE), (dict(kv_f32=1), SIZE), (dict(table_cols=1 << 27, table_stride=1 << 27), SIZE)]


@pytest.mark.parametrize("change,status", BAD_PAGES)
def test_bad_descriptions_are_refused(lib, change, status):
    assert rope(lib, pages(**change)) == status and b"ie_b200_rope_kv_paged" in lib.ie_b200_last_error()
    assert attn(lib, pages(**change)) == status and b"ie_b200_attn_decode_paged" in lib.ie_b200_last_error()


@pytest.mark.parametrize("change,status", [(dict(p=None), ARG), (dict(q=None), ARG), (dict(q_out=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(cos=None), ARG),
                                           (dict(sin=None), ARG), (dict(pos=None), ARG), (dict(q=AT + 2), ARG), (dict(seq=AT + 1), ARG), (dict(stride=48 * 512 + 2), ARG),
                                           (dict(nq=70000), SIZE), (dict(T=2, stride=1024), SIZE), (dict(T=2, out_stride=1024), SIZE)])
def test_rope_kv_paged_refuses(lib, change, status):
    assert rope(lib, **{"p": pages(), **change}) == status and b"ie_b200_rope_kv_paged" in lib.ie_b200_last_error()


@pytest.mark.parametrize("change,status", [(dict(p=None), ARG), (dict(q=None), ARG), (dict(out=None), ARG), (dict(lens=None), ARG), (dict(scratch=None), ARG),
                                           (dict(q=AT + 4), ARG), (dict(q_stride=4096 * 4 + 4), ARG), (dict(out=AT + 2), ARG), (dict(oq=AT + 1), ARG), (dict(lens=AT + 2), ARG),
                                           (dict(scratch=AT + 8), ARG), (dict(p=pages(page=8, page_stride=1 << 20)), SIZE), (dict(p=pages(page=24, page_stride=1 << 20)), SIZE),
                                           (dict(p=pages(hd=96)), SIZE), (dict(n_head=30), SIZE), (dict(n_head=0), SIZE), (dict(R=2, q_stride=1024), SIZE),
                                           (dict(R=2, out_stride=1024), SIZE), (dict(R=2, oq=AT, oq_stride=1024), SIZE), (dict(R=(1 << 20) + 1), SIZE),
                                           (dict(p=pages(n_kv=2048, page=1 << 20, table_cols=2000, table_stride=2000, page_stride=1 << 42), n_head=2048, q_stride=1 << 20, out_stride=1 << 20), SIZE)])
def test_attn_decode_paged_refuses(lib, change, status):
    assert attn(lib, **{"p": pages(), **change}) == status and b"ie_b200_attn_decode_paged" in lib.ie_b200_last_error()


def test_no_rows_is_no_launch(lib):
    before = lib.ie_b200_launch_count()
    assert rope(lib, pages(), T=0) == 0 and attn(lib, pages(), R=0) == 0
    assert lib.ie_b200_launch_count() == before


def test_wrappers_refuse_what_is_not_on_a_gpu():
    kp = torch.zeros(2, 1, 16, 32, dtype=torch.half)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="kp"):
        K.rope_kv_paged(torch.zeros(1, 96), kp, kp, table, torch.zeros(4, 16), torch.zeros(4, 16), one, None, 1, 1, 32, False)
    with pytest.raises(ValueError, match="kp"):
        K.attn_decode_paged(torch.zeros(1, 32), kp, kp, table, one, 1, None)


def sample(lib, x=AT, n=1000, idx=AT, prob=AT, u=AT, temp=None, k=None, p=None, m=None, T=1, x_stride=4000):
    return lib.ie_b200_sample(x, n, idx, prob, u, temp, k, p, m, T, x_stride, None)


@pytest.mark.parametrize("change,status", [(dict(x=None), ARG), (dict(idx=None), ARG), (dict(u=None), ARG), (dict(prob=AT + 2), ARG), (dict(x=AT + 1), ARG), (dict(temp=AT + 2), ARG), (dict(k=AT + 2), ARG),
                                           (dict(p=AT + 1), ARG), (dict(m=AT + 3), ARG), (dict(T=2, x_stride=4002), ARG), (dict(n=0), SIZE), (dict(n=360449), SIZE),
                                           (dict(T=2, x_stride=3996), SIZE), (dict(T=(1 << 20) + 1), SIZE)])
def test_sample_refuses(lib, change, status):
    assert sample(lib, **change) == status and b"ie_b200_sample" in lib.ie_b200_last_error()


def test_sample_no_rows(lib):
    before = lib.ie_b200_launch_count()
    assert sample(lib, T=0) == 0 and lib.ie_b200_launch_count() == before
    with pytest.raises(ValueError, match="x"):
        K.sample(torch.zeros(1, 10), torch.zeros(1))


def test_fill_is_refused_beyond_its_outputs(lib):
    assert lib.ie_b200_rope_kv_paged_fill(AT, AT, AT, AT, pages(), AT, AT, 80, AT, None, 32, 0, 1, 48 * 512, 32 * 512, None, 2, None) == ARG
    assert b"ie_b200_rope_kv_paged_fill" in lib.ie_b200_last_error()
    assert lib.ie_b200_attn_decode_paged_fill(AT, pages(), AT, None, AT, None, 32, 1, 4096 * 4, 4096 * 4, 5120, AT, None, 4, None) == ARG
    assert b"ie_b200_attn_decode_paged_fill" in lib.ie_b200_last_error()
