"""The 8-bit KV and sampling entry points refuse bad arguments on the host, before
anything is launched, and the definitions they are tested against hold where they
can be checked by hand."""
import math

import numpy as np
import pytest
import torch

from custom_inference_engine_b200 import native
from oracle import kv_q8 as ref
from oracle.sampling import sample_row

P = 1 << 20


def _call(name, base, **kw):
    base.update(kw)
    return getattr(native.lib(), name)(*base.values())


def _pool():
    return dict(hkv=2, d=64, page=16)


def _tail():
    return dict(n_pages=10, n_slots=3, bt_stride=10, pstride=2048, hstride=1024)


def decode_update(**kw):
    return _call("cie_kv_q8_decode_update", dict(
        k=P, v=P, s=P, lens=P, slots=P, bt=P, kn=P, vn=P, batch=2, **_pool(), **_tail(),
        kt=1152, kh=64, vt=1152, vh=64, stream=None), **kw)


def mixed_update(**kw):
    return _call("cie_kv_q8_mixed_update", dict(
        k=P, v=P, s=P, cu=P, kvl=P, slots=P, bt=P, kn=P, vn=P, batch=2, T=8, **_pool(),
        **_tail(), kt=1152, kh=64, vt=1152, vh=64, stream=None), **kw)


def rope_decode(**kw):
    return _call("cie_rope_kv_q8_decode_update", dict(
        qkv=P, qkv_tok=1152, cos=P, sin=P, cs_tok=64, q=P, k=P, v=P, s=P, lens=P, slots=P, bt=P,
        batch=2, hq=14, **_pool(), **_tail(), stream=None), **kw)


def rope_mixed(**kw):
    return _call("cie_rope_kv_q8_mixed_update", dict(
        qkv=P, qkv_tok=1152, cos=P, sin=P, cs_tok=64, q=P, k=P, v=P, s=P, cu=P, kvl=P, slots=P,
        bt=P, batch=2, T=8, hq=14, **_pool(), **_tail(), stream=None), **kw)


def read(**kw):
    return _call("cie_kv_q8_read", dict(
        k=P, v=P, s=P, starts=None, lens=P, slots=P, bt=P, ko=P, vo=P, batch=2, **_pool(),
        **_tail(), opage=2048, ohead=1024, stream=None), **kw)


def attend(**kw):
    return _call("cie_decode_attention_q8", dict(
        q=P, k=P, v=P, s=P, lens=P, slots=P, bt=P, o=P, ws=None, ws_bytes=0, batch=2, hq=14,
        **_pool(), **_tail(), splits=1, stream=None), **kw)


def sample(**kw):
    return _call("cie_sample_rows", dict(
        x=P, rows=2, vocab=100, stride=100, u=P, t=P, k=None, p=None, m=None, out=P,
        stream=None), **kw)


POOL_CASES = [(dict(k=None), -1), (dict(s=None), -1), (dict(d=128), -2), (dict(page=32), -2),
              (dict(hkv=0), -2), (dict(pstride=2000), -1), (dict(pstride=2056, hstride=1028), -4),
              (dict(k=P + 8), -4), (dict(s=P + 2), -4), (dict(n_pages=0), -1),
              (dict(bt=None), -1), (dict(slots=None), -1), (dict(batch=-1), -1)]


@pytest.mark.parametrize("call", [decode_update, mixed_update, rope_decode, rope_mixed, read,
                                  attend])
@pytest.mark.parametrize("kw,status", POOL_CASES, ids=lambda x: str(x))
def test_pool_checks(call, kw, status):
    assert call(**kw) == status
    assert native.lib().cie_last_error_message()


@pytest.mark.parametrize("call,kw,status", [
    (decode_update, dict(lens=None), -1), (decode_update, dict(kn=None), -1),
    (mixed_update, dict(cu=None), -1), (mixed_update, dict(kvl=None), -1),
    (mixed_update, dict(T=-1), -1), (mixed_update, dict(vn=None), -1),
    (rope_decode, dict(qkv=None), -1), (rope_decode, dict(qkv_tok=1100), -1),
    (rope_decode, dict(qkv_tok=1156), -4), (rope_decode, dict(cs_tok=32), -1),
    (rope_decode, dict(q=P + 2), -4), (rope_mixed, dict(hq=0), -1), (rope_mixed, dict(cos=None), -1),
    (read, dict(ko=None), -1), (read, dict(opage=1000), -1), (read, dict(vo=P + 2), -4),
    (read, dict(batch=65536), -2), (attend, dict(q=None), -1), (attend, dict(hkv=3, hq=21, pstride=4096), -2),
    (attend, dict(hq=18), -2), (attend, dict(hq=15), -2), (attend, dict(n_pages=1 << 31), -3),
    (attend, dict(splits=4), -5), (attend, dict(splits=4, ws=P, ws_bytes=100), -5),
    (attend, dict(splits=5000), -1), (attend, dict(o=P + 8), -4), (attend, dict(batch=65536), -2),
    (sample, dict(x=None), -1), (sample, dict(u=None), -1), (sample, dict(t=None), -1),
    (sample, dict(out=None), -1), (sample, dict(vocab=0), -1), (sample, dict(vocab=-1), -1),
    (sample, dict(rows=-1), -1), (sample, dict(stride=99), -1), (sample, dict(x=P + 1), -4),
    (sample, dict(vocab=524225, stride=524225), -2),
])
def test_argument_checks(call, kw, status):
    assert call(**kw) == status


def test_nothing_to_do():
    assert decode_update(batch=0, k=None) == 0 and mixed_update(T=0) == 0
    assert rope_decode(batch=0) == 0 and rope_mixed(T=0, qkv=None) == 0
    assert read(batch=0) == 0 and attend(batch=0, q=None) == 0 and sample(rows=0, x=None) == 0


def test_scale_of_a_page():
    """The smallest power of two that holds the largest value."""
    assert ref.page_scale(0.0) == 2.0 ** -24 and ref.page_scale(127.0) == 1.0
    assert ref.page_scale(127.0625) == 2.0 and ref.page_scale(63.5) == 0.5
    assert ref.page_scale(65504.0) == 512.0 and ref.page_scale(math.inf) == 512.0


def test_sampling_definition_by_hand():
    x = np.log([0.5, 0.25, 0.125, 0.125])[[3, 0, 2, 1]]  # tokens 1, 3, then 0 and 2 tied
    at = lambda u, **kw: sample_row(x, u, 1.0, **kw)
    assert [at(u) for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.87, 0.88, 0.99)] == [1, 1, 3, 3, 0, 0, 2, 2]
    assert [at(u, top_k=2) for u in (0.0, 0.66, 0.67, 0.99)] == [1, 1, 3, 3]
    assert [at(u, top_p=0.6) for u in (0.66, 0.67)] == [1, 3]
    assert at(0.99, top_p=0.5 - 1e-9) == 1 and at(0.99, min_p=0.3) == 3 and at(0.99, top_k=3) == 0
    assert sample_row([0.0, 2.0, 2.0], 0.99, 0.0) == 1
    assert sample_row([-math.inf] * 3, 0.5, 1.0) == 0
