"""Argument checks of the attention-step entry points: every refusal comes from
the host before any CUDA call, so the addresses here are never used."""
import ctypes

import pytest

import kvmret

lib = kvmret.lib
A = 4096  # an aligned address that nothing reads


def qk_args(**kw):
    a = dict(q_dev=A, k_dev=A, q_stride=1024, k_stride=256, q_weight_dev=None, k_weight_dev=None,
             pos_dev=A, q_rot_dev=A, k_rot_dev=A, q_raw_dev=None, k_raw_dev=None, n_tok=2,
             n_head=8, n_head_kv=2, d_head=128, n_rot=128, fwht_n=0, type=kvmret.TYPE_F16,
             eps=1e-6, freq_base=1e6, freq_scale=1.0)
    a.update(kw)
    return kvmret.QkArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(d_head=96, n_rot=96), b"d_head"), (dict(n_rot=64), b"n_rot"), (dict(fwht_n=64), b"fwht_n"),
    (dict(type=8), b"type"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(freq_base=0.0), b"freq_base"), (dict(freq_scale=float("inf")), b"freq_base"),
    (dict(pos_dev=None), b"positions"), (dict(q_dev=None), b"without its rows"),
    (dict(n_head=0), b"heads"), (dict(q_stride=1016), b"overlap"), (dict(k_stride=0), b"overlap"),
    (dict(q_dev=A + 2), b"aligned"), (dict(q_stride=1028), b"aligned"),
    (dict(k_rot_dev=A + 8), b"aligned"), (dict(type=kvmret.TYPE_F32, q_stride=1026), b"aligned"),
])
def test_qk_norm_rope_refuses(kw, word):
    assert lib.kvmret_qk_norm_rope(ctypes.byref(qk_args(**kw)), None) == -1
    assert word in lib.kvmret_last_error()


def test_qk_norm_rope_nothing_to_do():
    assert lib.kvmret_qk_norm_rope(None, None) == -1
    assert lib.kvmret_qk_norm_rope(ctypes.byref(qk_args(n_tok=0, pos_dev=None)), None) == 0
    assert lib.kvmret_qk_norm_rope(ctypes.byref(qk_args(q_rot_dev=None, k_rot_dev=None)), None) == 0


def pages_desc(**kw):
    a = dict(k_dev=A, v_dev=A, k_page_bytes=0, v_page_bytes=0, n_pages=4, page_tokens=32,
             n_head_kv=2, d_head=128, k_type=kvmret.TYPE_F16, v_type=kvmret.TYPE_F16)
    a.update(kw)
    return kvmret.PagesDesc(**a)


BAD_PAGES = [
    (dict(k_dev=None), b"null"), (dict(d_head=80), b"d_head"), (dict(n_head_kv=0), b"n_head_kv"),
    (dict(n_pages=0), b"pages"), (dict(page_tokens=0), b"pages"),
    (dict(n_pages=1 << 20, page_tokens=1 << 12), b"pages"), (dict(k_type=3), b"type"),
    (dict(v_type=0), b"type"), (dict(k_type=kvmret.TYPE_Q8_0, n_head_kv=1), b"row bytes"),
    (dict(k_dev=A + 8), b"aligned"), (dict(v_page_bytes=32 * 512 + 8), b"aligned"),
    (dict(k_page_bytes=31 * 512), b"shorter"),
]


@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_paged_append_refuses_pages(kw, word):
    rc = lib.kvmret_paged_append(ctypes.byref(pages_desc(**kw)), A, 0, A, 0, A, A, 3, 1e6, 1.0, 0,
                                 None)
    assert rc == -1 and word in lib.kvmret_last_error()


@pytest.mark.parametrize("args,word", [
    ((None, 0, A, 0, A, A, 3, 1e6, 1.0, 0), b"null"), ((A, 0, A, 0, None, A, 3, 1e6, 1.0, 0), b"null"),
    ((A, 0, A, 0, A, A, 3, 1e6, 1.0, 64), b"fwht_n"), ((A, 0, A, 0, A, A, 3, 0.0, 1.0, 0), b"freq"),
    ((A + 2, 0, A, 0, A, A, 3, 1e6, 1.0, 0), b"aligned"),
    ((A, 260, A, 0, A, A, 3, 1e6, 1.0, 0), b"aligned"),
    ((A, 0, A, 248, A, A, 3, 1e6, 1.0, 0), b"overlap"),
])
def test_paged_append_refuses(args, word):
    rc = lib.kvmret_paged_append(ctypes.byref(pages_desc()), *args, None)
    assert rc == -1 and word in lib.kvmret_last_error()


def test_paged_append_of_no_tokens():
    assert lib.kvmret_paged_append(ctypes.byref(pages_desc()), None, 0, None, 0, None, None, 0, 1e6,
                                   1.0, 0, None) == 0
